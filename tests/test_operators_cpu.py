"""The operators' 64-bit forms against differences and published values, and the refusals that
need no GPU."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import operator_forms as forms
import persistent_lstm_hip_b200 as plstm
from persistent_lstm_hip_b200 import _lib

D = torch.float64


def _differences(fn, x, v, h=1e-6):
    return (fn(x + h * v) - fn(x - h * v)) / (2 * h)


def _randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + 17 * len(shape)), dtype=D)


# Central differences at h = 1e-6 in f64 of sums of O(100) terms: 1e-16 * 100 / 1e-6 = 1e-8.
DIFF_TOL = 2e-7


@pytest.mark.parametrize("lengths", [None, [0, 5, 9]])
def test_scan_gradient_formula_against_differences(lengths):
    B, T, H = 3, 9, 4
    gates, c0, dh, dc_n = _randn(B, T, 4 * H), _randn(B, H, seed=1), _randn(B, T, H, seed=2), _randn(B, H, seed=3)
    lens = None if lengths is None else torch.tensor(lengths)

    def loss(gates, c0):
        s = forms.scan_forward(gates, c0, lens)
        return float((s["h"] * dh).sum() + (s["c_n"] * dc_n).sum())

    r = forms.scan_backward(forms.scan_forward(gates, c0, lens), dh, dc_n)
    for k in range(3):
        v, u = _randn(B, T, 4 * H, seed=10 + k), _randn(B, H, seed=20 + k)
        assert abs(_differences(lambda x: loss(x, c0), gates, v) - float((r["dgates"] * v).sum())) < DIFF_TOL
        assert abs(_differences(lambda x: loss(gates, x), c0, u) - float((r["dc0"] * u).sum())) < DIFF_TOL


def test_norm_gradient_formula_against_differences():
    M, N, eps = 5, 7, 1e-5
    x, w, b, dy, dz = _randn(M, N), _randn(N, seed=1), _randn(N, seed=2), _randn(M, N, seed=3), _randn(M, N, seed=4)

    def loss(x, w, b):
        return float((forms.norm_forward(x, w, b, eps)["y"] * dy).sum() + (x * dz).sum())

    r = forms.norm_backward(forms.norm_forward(x, w, b, eps), dy, dz)
    for k in range(3):
        v, u = _randn(M, N, seed=10 + k), _randn(N, seed=20 + k)
        assert abs(_differences(lambda a: loss(a, w, b), x, v) - float((r["dv"] * v).sum())) < DIFF_TOL
        assert abs(_differences(lambda a: loss(x, a, b), w, u) - float((r["dw"] * u).sum())) < DIFF_TOL
        assert abs(_differences(lambda a: loss(x, w, a), b, u) - float((r["db"] * u).sum())) < DIFF_TOL


def test_philox_known_answers():
    """The known-answer vectors that the generator's authors publish with it."""
    f = 0xFFFFFFFF
    assert forms.philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert forms.philox([f] * 4, [f] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert forms.philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_keep_mask_is_philox():
    seed, offset, p = 0x123456789ABCDEF, 0xFEDCBA9876543210, 0.3
    at = np.array([0, 1, 6, 4 * (1 << 32) + 11, (1 << 62) + 3], dtype=np.uint64)
    keep = forms.keep_mask(at, p, seed, offset)
    for e, k in zip(at.tolist(), keep.tolist()):
        b = e // 4
        w = forms.philox([b & 0xFFFFFFFF, b >> 32, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32])
        assert k == (w[e % 4] >= int(p * 2 ** 32))


# ---- refusals of the C ABI (before any CUDA call) -------------------------------------------------------
def _scan_desc(**kw):
    base = dict(batch=2, seq_len=3, hidden=4, dtype=_lib.F32, device=0, reserved=0, gates_batch_stride=48,
                gates_time_stride=16, h_batch_stride=12, h_time_stride=4, dgates_batch_stride=48,
                dgates_time_stride=16)
    base.update(kw)
    return _lib.ScanDesc(*[base[f] for f, _ in _lib.ScanDesc._fields_])


@pytest.mark.parametrize("bad, msg", [
    (dict(batch=-1), "batch"), (dict(seq_len=-1), "seq_len"), (dict(seq_len=2**31 - 1), "seq_len"),
    (dict(hidden=0), "hidden"), (dict(dtype=5), "dtype"), (dict(reserved=1), "reserved"),
    (dict(gates_time_stride=-16), "strides"),
])
def test_scan_descriptor_refusals(bad, msg):
    lib, n = _lib.load(), ctypes.c_size_t(0)
    d = _scan_desc(**bad)
    for rc in (lib.plstm_gated_scan_checkpoint_size(ctypes.byref(d), ctypes.byref(n)),
               lib.plstm_gated_scan_forward(ctypes.byref(d), 16, None, None, 16, 16, None, None),
               lib.plstm_gated_scan_backward(ctypes.byref(d), 16, None, 16, 16, None, 16, None, None)):
        assert rc == _lib.EINVAL and msg in _lib.last_error()


def test_scan_pointer_refusals():
    lib, d = _lib.load(), ctypes.byref(_scan_desc())
    for args, msg in (((None, None, None, 16, 16, None), "gates and h"), ((16, None, None, None, 16, None), "gates and h"),
                      ((16, None, None, 16, None, None), "c_n"), ((18, None, None, 16, 16, None), "aligned"),
                      ((16, 2, None, 16, 16, None), "aligned")):
        assert lib.plstm_gated_scan_forward(d, *args, None) == _lib.EINVAL and msg in _lib.last_error()
    assert lib.plstm_gated_scan_backward(d, 16, None, None, 16, None, 16, None, None) == _lib.EINVAL
    assert "checkpoints" in _lib.last_error()
    n = ctypes.c_size_t(0)
    assert lib.plstm_gated_scan_checkpoint_size(ctypes.byref(_scan_desc(seq_len=9)), ctypes.byref(n)) == 0
    assert n.value == 2 * 2 * 4 * 4  # ceil(9 / 8) segments


def _norm_desc(**kw):
    base = dict(rows=4, cols=8, x_dtype=_lib.F16, z_dtype=_lib.F16, w_dtype=_lib.F32, device=0, eps=1e-5, x_stride=8,
                residual_stride=8, dy_stride=8, dz_stride=8)
    base.update(kw)
    return _lib.NormDesc(*[base[f] for f, _ in _lib.NormDesc._fields_])


@pytest.mark.parametrize("bad, msg", [
    (dict(rows=-1), "rows"), (dict(cols=0), "cols"), (dict(cols=_lib.NORM_MAX_COLS + 1), "cols"),
    (dict(x_dtype=3), "dtype"), (dict(z_dtype=_lib.BF16), "z_dtype"), (dict(w_dtype=_lib.BF16), "w_dtype"),
    (dict(eps=-1.0), "eps"), (dict(x_stride=-8), "strides"),
])
def test_norm_descriptor_refusals(bad, msg):
    lib, d = _lib.load(), ctypes.byref(_norm_desc(**bad))
    assert lib.plstm_layer_norm_forward(d, None, 16, 16, None, None, 16, 16, None, None) == _lib.EINVAL
    assert msg in _lib.last_error()
    assert lib.plstm_layer_norm_backward(d, None, 1, 16, None, 16, None, 16, 16, None, None, None, None, 0,
                                         None) == _lib.EINVAL
    assert msg in _lib.last_error()


def test_norm_call_refusals():
    lib, d, drop = _lib.load(), ctypes.byref(_norm_desc()), ctypes.byref(_lib.DropoutDesc(0.5, 1, 0, None))
    assert lib.plstm_layer_norm_forward(d, drop, 16, None, None, None, None, 16, None, None) == _lib.EINVAL
    assert "residual" in _lib.last_error()
    assert lib.plstm_layer_norm_forward(d, None, 16, 16, None, None, None, 16, None, None) == _lib.EINVAL
    f32z = ctypes.byref(_norm_desc(z_dtype=_lib.F32))
    assert lib.plstm_layer_norm_forward(f32z, None, 16, None, None, None, None, 16, None, None) == _lib.EINVAL
    assert lib.plstm_layer_norm_backward(d, None, 1, 16, None, 16, None, 16, 16, None, 16, None, 16, 8,
                                         None) == _lib.EWORKSPACE
    assert lib.plstm_layer_norm_backward(d, None, 0, 16, 16, 16, None, 16, 16, None, None, None, None, 0,
                                         None) == _lib.EINVAL


@pytest.mark.parametrize("p", [-0.1, 1.1, float("nan")])
def test_dropout_refuses_p(p):
    lib, d = _lib.load(), _lib.DropoutDesc(p, 1, 0, None)
    assert lib.plstm_dropout(ctypes.byref(d), 4, 16, _lib.F32, None, 16, _lib.F32, 0, None) == _lib.EINVAL
    assert "p must be" in _lib.last_error()


def test_dropout_call_refusals():
    lib, d = _lib.load(), ctypes.byref(_lib.DropoutDesc(0.5, 1, 0, None))
    for args in ((-1, 16, _lib.F32, None, 16, _lib.F32), (4, None, _lib.F32, None, 16, _lib.F32),
                 (4, 16, _lib.F16, None, 16, _lib.BF16), (4, 18, _lib.F32, None, 16, _lib.F32),
                 (4, 16, 9, None, 16, _lib.F32)):
        assert lib.plstm_dropout(d, *args, 0, None) == _lib.EINVAL


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 8)
    for call in (lambda: plstm.gated_scan(x), lambda: plstm.layer_norm(x), lambda: plstm.dropout(x, 0.5, 1),
                 lambda: plstm.dropout_add_layer_norm(x, x), lambda: plstm.gated_scan_step(x[0], x[0, :, :2])):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()
