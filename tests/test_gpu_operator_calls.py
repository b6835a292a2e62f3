"""The training and streaming operators' calls on the GPU: what autograd, hooks, tracers and threads
see of them."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import operator_forms as forms
import persistent_lstm_hip_b200 as plstm

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _randn(*shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + 31 * len(shape))).to("cuda:0", dtype)


# ---- a tensor seed under saved-tensor hooks ----------------------------------------------------------
@pytest.mark.parametrize("fused", [False, True])
def test_temporary_seed_under_a_checkpoint(cuda_device, fused):
    """The seed is made inside the checkpointed function and freed before the backward: the mask of
    the gradients is the forward's all the same."""
    n, p = 4096, 0.5
    base = torch.tensor([41], device=cuda_device)

    def call(x):
        if fused:
            return plstm.dropout_add_layer_norm(x, torch.zeros_like(x), None, None, p, base + 1)[1]
        return plstm.dropout(x, p, base + 1)

    x = _randn(8, n // 8).requires_grad_(True)
    y = checkpoint(call, x, use_reentrant=False)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(x))
    keep = forms.keep_mask(np.arange(n), p, 42, 0).view(8, n // 8)
    assert torch.equal(y.detach().cpu() != 0, keep)
    assert torch.equal(dx.cpu(), keep.float() * 2)


def test_seed_advanced_under_hooks_that_copy(cuda_device):
    x, seed = _randn(1000).requires_grad_(True), torch.tensor([42], device=cuda_device)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t):
        y = plstm.dropout(x, 0.5, seed)
    seed.add_(1)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(x))
    assert torch.equal(dx.cpu(), forms.keep_mask(np.arange(1000), 0.5, 42, 0).float() * 2)


# ---- lengths --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dev", ["cuda:0", "cpu"])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16,
                                   torch.uint32, torch.uint64, torch.bool])
def test_lengths_of_any_type_are_clamped_not_wrapped(cuda_device, dtype, dev):
    B, T, H = 4, 300, 8
    top = 1 if dtype is torch.bool else torch.iinfo(dtype).max
    values = [0, 1, top, min(top, 2 ** 32 + 5)]
    gates, c0 = _randn(B, T, 4 * H), _randn(B, H)
    want = plstm.gated_scan(gates, c0, torch.tensor([min(v, T) for v in values], dtype=torch.int32))
    got = plstm.gated_scan(gates, c0, torch.tensor(values, dtype=dtype).to(dev))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_lengths_below_int32_are_zero(cuda_device):
    gates, c0 = _randn(2, 9, 16), _randn(2, 4)
    h, c_n = plstm.gated_scan(gates, c0, torch.tensor([-(2 ** 31) - 7, torch.iinfo(torch.int64).min]))
    assert (h == 0).all() and torch.equal(c_n, c0)


# ---- writes into the caller's state --------------------------------------------------------------------
def test_streaming_from_a_state_whose_graph_is_still_needed(cuda_device):
    """The regressor's states are attached to its graph; streaming on from them in place and then
    differentiating is an error, never a gradient with the new values."""
    torch.manual_seed(0)
    m = plstm.GatedScanRegressor(3, 16, 2, 2).to(cuda_device)
    _, state = m(_randn(2, 7, 3))
    loss = (state[0] ** 2).sum()
    m.step(_randn(2, 3), state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    _, state = m(_randn(2, 7, 3))
    loss = (state[0] ** 2).sum()
    m.step(_randn(2, 3), [c.detach().clone() for c in state])
    loss.backward()


def test_step_in_inference_mode(cuda_device):
    gates = _randn(2, 16)
    with torch.inference_mode():
        c = torch.zeros(2, 4, device=cuda_device)
        h, _ = plstm.gated_scan_step(gates, c, out_c=c)
    want_h, want_c = plstm.gated_scan_step(gates, torch.zeros(2, 4, device=cuda_device))
    assert torch.equal(h, want_h) and torch.equal(c, want_c)


# ---- in-place operations on results -----------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(16,), (4, 16), (2, 3, 16), (3, 0, 16)])
def test_in_place_operations_on_results(cuda_device, shape):
    x, w, res = _randn(*shape).requires_grad_(True), _randn(16, seed=1).requires_grad_(True), _randn(*shape, seed=2)
    for call in (lambda: plstm.layer_norm(x, w), lambda: plstm.dropout_add_layer_norm(x, res, w, None, 0.25, 3)[0],
                 lambda: plstm.dropout(x, 0.25, 3) * w):
        want = call().relu()
        got = call().relu_()
        assert got.shape == shape and torch.equal(got, want)
        grads = [torch.autograd.grad(y, (x, w), torch.ones_like(y)) for y in (got, want)]
        assert all(torch.equal(a, b) for a, b in zip(*grads))
