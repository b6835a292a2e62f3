"""Trainable gated-scan layers: LSTM-like layers whose gates do not look back, so time is
scanned in parallel, with their streaming form.

* ``GatedScanLayer``: nn.LSTM-style projection (weight_ih [4H, I], bias [4H], gate order
  i, f, g, o) followed by ``gated_scan``.
* ``GatedScanRegressor``: a pre-norm residual stack of such layers with a Linear head,
  x [B,T,I] -> [B,T,O]; ``step`` advances a batch of streams by one time step.

The projections are plain library GEMMs (nn.Linear); everything else is this package's kernels.
"""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops


class GatedScanLayer(nn.Module):
    """x [B,T,I] -> (h [B,T,H], c_n [B,H] f32); the state is only ever the cell c."""

    def __init__(self, input_size: int, hidden_size: int, forget_bias: float = 1.0):
        super().__init__()
        self.input_size, self.hidden_size = input_size, hidden_size
        self.weight_ih = nn.Parameter(torch.empty(4 * hidden_size, input_size))
        self.bias = nn.Parameter(torch.zeros(4 * hidden_size))
        nn.init.uniform_(self.weight_ih, -1 / math.sqrt(input_size), 1 / math.sqrt(input_size))
        with torch.no_grad():
            self.bias[hidden_size:2 * hidden_size] = forget_bias

    def forward(self, x: torch.Tensor, c0: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        return ops.gated_scan(F.linear(x, self.weight_ih, self.bias), c0, lengths)

    @torch.no_grad()
    def step(self, x: torch.Tensor, c: torch.Tensor) -> torch.Tensor:
        """x [B,I] -> h [B,H]; advances c [B,H] in place."""
        return ops.gated_scan_step(F.linear(x, self.weight_ih, self.bias), c, out_c=c)[0]


class GatedScanRegressor(nn.Module):
    """Linear(I, H), then per layer norm -> GatedScanLayer -> Linear(H, H) -> dropout + residual,
    then norm -> Linear(H, O).  Each residual step is one kernel with the norm that follows it."""

    def __init__(self, input_dim: int, hidden_dim: int, output_dim: int, n_layers: int, dropout: float = 0.2,
                 eps: float = 1e-5):
        super().__init__()
        self.dropout, self.eps, self.hidden_dim = dropout, eps, hidden_dim
        self.embed = nn.Linear(input_dim, hidden_dim)
        self.layers = nn.ModuleList(GatedScanLayer(hidden_dim, hidden_dim) for _ in range(n_layers))
        self.outs = nn.ModuleList(nn.Linear(hidden_dim, hidden_dim) for _ in range(n_layers))
        self.norm_weight = nn.ParameterList(nn.Parameter(torch.ones(hidden_dim)) for _ in range(n_layers + 1))
        self.norm_bias = nn.ParameterList(nn.Parameter(torch.zeros(hidden_dim)) for _ in range(n_layers + 1))
        self.linear = nn.Linear(hidden_dim, output_dim)

    def init_state(self, batch: int) -> List[torch.Tensor]:
        dev = self.linear.weight.device
        return [torch.zeros(batch, self.hidden_dim, device=dev, dtype=torch.float32) for _ in self.layers]

    def _blocks(self, z, scan, p, seed):
        y = ops.layer_norm(z, self.norm_weight[0], self.norm_bias[0], self.eps)
        for l, (layer, out) in enumerate(zip(self.layers, self.outs)):
            y, z = ops.dropout_add_layer_norm(out(scan(l, layer, y)), z, self.norm_weight[l + 1],
                                              self.norm_bias[l + 1], p, seed, l, eps=self.eps)
        return self.linear(y)

    def forward(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None,
                state: Optional[List[torch.Tensor]] = None, seed=None) -> Tuple[torch.Tensor, List[torch.Tensor]]:
        """x [B,T,I] -> (out [B,T,O], state after each row's last step, one c [B,H] f32 per layer).

        seed: the dropout seed of this pass in training mode (drawn from torch's CPU generator by
        default); layer l draws at offset l.  Outputs past a row's length are not meaningful.
        """
        p = self.dropout if self.training else 0.0
        if seed is None:
            seed = int(torch.randint(1 << 62, ())) if p > 0 else 0
        if lengths is not None:  # once for all layers
            lengths = ops.lengths32(lengths, x.shape[0], x.shape[1], x.device)
        state_n = []

        def scan(l, layer, y):
            h, c_n = layer(y, None if state is None else state[l], lengths)
            state_n.append(c_n)
            return h

        return self._blocks(self.embed(x), scan, p, seed), state_n

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: List[torch.Tensor]) -> torch.Tensor:
        """x [B,I] -> out [B,O] for the next time step of B streams; advances `state` in place."""
        return self._blocks(self.embed(x), lambda l, layer, y: layer.step(y, state[l]), 0.0, 0)
