"""The training and streaming operators on the GPU where f32's range ends, against their 64-bit forms."""
from __future__ import annotations

import pytest
import torch

import operator_forms as forms
from operator_forms import f64
from test_gpu_operators import _check_scan, _gates, _randn
import persistent_lstm_hip_b200 as plstm

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# ---- products of a closed gate and a saturated tanh ---------------------------------------------------
def _closed_gates(B, T, H, dtype, dev):
    """Input and output gates between -64 and -85 over candidates from -20 to 20: products from 1e-28 down to
    1e-37, which f32 and bf16 hold."""
    gates = _gates(B, T, H, F32, "cpu", seed=4)
    gates[..., :H] = -torch.linspace(64, 85, H)
    gates[..., 2 * H:3 * H] = torch.linspace(-20, 20, B * T).view(B, T, 1)
    gates[..., 3 * H:] = -torch.linspace(85, 64, H)
    return gates.to(dev, dtype)


@pytest.mark.parametrize("B,T,H", [(3, 1, 24), (3, 3, 24), (2, 40, 24), (2, 40, 23)])
@pytest.mark.parametrize("c0", [0.0, -20.0, 20.0])
def test_closed_gates_over_saturated_candidates(cuda_device, B, T, H, c0):
    d = cuda_device
    _check_scan(_closed_gates(B, T, H, F32, d), torch.full((B, H), c0, device=d), None,
                _randn(B, T, H, dtype=F32, dev=d), _randn(B, H, dtype=F32, dev=d, seed=1))


@pytest.mark.parametrize("T,H", [(1, 24), (3, 24), (40, 24), (40, 23)])
def test_closed_gates_in_16_bits(cuda_device, T, H):
    """The exponential of a 16-bit gate x carries |x| units in 2^-24 (the rounding of its argument) on top of about ten
    of the functions around it: 95 units for |x| <= 85.  A step's forget gate and sum add up to five: 200 over 40 steps.
    Where all terms have one sign that is below 2^-15 of the state.  The output adds its own rounding, 2^-8 of its
    size."""
    gates = _closed_gates(2, T, H, BF16, cuda_device)
    gates[..., 2 * H:3 * H] = -gates[..., 2 * H:3 * H].abs() - 1
    h, c_n = plstm.gated_scan(gates)
    s = forms.scan_forward(f64(gates))
    assert ((f64(c_n) - s["c_n"]).abs() <= 2.0 ** -15 * s["c_n"].abs()).all()
    h_up, _ = plstm.gated_scan(gates, torch.full((2, H), -20.0, device=cuda_device))
    s = forms.scan_forward(f64(gates), torch.full((2, H), -20.0, dtype=torch.float64))
    assert ((f64(h_up) - s["h"]).abs() <= 2.0 ** -7 * s["h"].abs() + 2.0 ** -126).all()


# ---- norm without eps of rows whose variance is subnormal -----------------------------------------------
@pytest.mark.parametrize("k", [0, 1, 2, 3])
def test_norm_of_a_subnormal_variance(cuda_device, k):
    """Rows whose mean, squares and variance (2^k of f32's smallest step) are exact: what is left is the reciprocal
    square root and two products, a few units in 2^-24."""
    n, a = 16 >> k, 2.0 ** -73
    x = torch.zeros(1, n)
    x[0, 0], x[0, 1] = a, -a
    var = 2 * a * a / n
    assert var == 2.0 ** (k - 149)
    y = plstm.layer_norm(x.to(cuda_device), eps=0.0)
    want = x.double() / var ** 0.5
    assert ((f64(y) - want).abs() <= 16 * 2.0 ** -24 * want.abs()).all()
