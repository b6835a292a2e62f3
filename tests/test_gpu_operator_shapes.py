"""The training and streaming operators on the GPU at sizes that reach every split of the work: several rows a
team, two and four chunks a thread with and without phases, short and single-step scans, warps that walk their
rows alone."""
from __future__ import annotations

import threading

import pytest
import torch

import operator_forms as forms
from operator_forms import assert_within, f64
from test_gpu_operators import FUSED_TYPES, _check_norm, _check_scan, _gates, _norm_inputs, _randn, test_fused_step as \
    check_fused_step
import persistent_lstm_hip_b200 as plstm

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("B,T,H", [(5, 2, 64), (7, 3, 33), (300, 4, 64),  # one segment of up to four steps
                                   (300, 1, 64), (5, 1, 3),              # one step, backward too
                                   (2500, 40, 64), (1300, 21, 33),       # time is not split, several turns
                                   (1, 6001, 21), (3, 3001, 255)])       # clusters over single channels
def test_scan_splits(cuda_device, dtype, ragged, B, T, H):
    d = cuda_device
    lens = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(5)).to(d) if ragged else None
    _check_scan(_gates(B, T, H, dtype, d), _randn(B, H, dtype=F32, dev=d), lens, _randn(B, T, H, dtype=dtype, dev=d),
                _randn(B, H, dtype=F32, dev=d, seed=1))


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("M,N", [(5003, 1001), (257, 2050), (3001, 2056), (20011, 129)])
def test_norm_splits(cuda_device, dtype, wdtype, M, N):
    _check_norm(*_norm_inputs(M, N, dtype, wdtype, cuda_device))


@pytest.mark.parametrize("dtype,rdtype,wdtype", FUSED_TYPES)
@pytest.mark.parametrize("M,N", [(20011, 512), (3001, 2056), (20011, 129), (5003, 1001)])
def test_fused_splits(cuda_device, dtype, rdtype, wdtype, M, N):
    check_fused_step(cuda_device, dtype, rdtype, wdtype, M, N, 0.3)


@pytest.mark.parametrize("rdtype", [F32, BF16])
def test_fused_residual_stream_has_the_dropouts_bits_at_any_alignment(cuda_device, rdtype):
    """z is the separate dropout's bit for bit, whatever the offsets; y is the norm of that z."""
    d, (M, N) = cuda_device, (37, 1024)
    wide, res = _randn(M, N + 9, dtype=BF16, dev=d), _randn(M, N + 9, dtype=rdtype, dev=d, seed=1)
    for i, j in ((0, 0), (1, 0), (0, 3), (1, 8)):
        x, r = wide[:, i:i + N], res[:, j:j + N]
        y, z = plstm.dropout_add_layer_norm(x, r, p=0.3, seed=5)
        assert torch.equal(z, plstm.dropout(x, 0.3, 5, residual=r))
        s = forms.norm_forward(f64(z), None, None, 1e-5)
        assert_within(y, s["y"], s["y_err"], "y")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,H", [(1, 1), (3, 17), (40, 64)])
def test_step_gradients(cuda_device, dtype, B, H):
    """A step outside no_grad is differentiable: the gradients of a scan of one step."""
    d = cuda_device
    gates, c = _gates(B, 1, H, dtype, d)[:, 0], _randn(B, H, dtype=F32, dev=d)
    dh, dc = _randn(B, H, dtype=dtype, dev=d, seed=1), _randn(B, H, dtype=F32, dev=d, seed=2)
    g, c_in = gates.clone().requires_grad_(True), c.clone().requires_grad_(True)
    h, c_n = plstm.gated_scan_step(g, c_in)
    dg, dc0 = torch.autograd.grad((h, c_n), (g, c_in), (dh, dc))
    s = forms.scan_forward(f64(gates)[:, None], f64(c))
    r = forms.scan_backward(s, f64(dh)[:, None], f64(dc))
    assert_within(h, s["h"][:, 0], s["h_err"][:, 0], "h")
    assert_within(c_n, s["c_n"], s["c_n_err"], "c_n")
    assert_within(dg, r["dgates"][:, 0], r["dgates_err"][:, 0], "dgates")
    assert_within(dc0, r["dc0"], r["dc0_err"], "dc0")


def test_norms_of_other_shapes_on_other_threads(cuda_device):
    """Threads that launch shapes with different shared memory at the same time do not take it from one another."""
    shapes = [(33, 64), (40, 4096), (17, 16384), (600, 512), (9, 129), (5, 8192)]
    inputs = [(_randn(M, N, dtype=F32, dev=cuda_device, seed=k), _randn(N, dtype=F32, dev=cuda_device, seed=k),
               _randn(M, N, dtype=F32, dev=cuda_device, seed=50 + k)) for k, (M, N) in enumerate(shapes)]
    streams = [torch.cuda.Stream() for _ in shapes]

    def call(k):
        x, w, dy = inputs[k]
        with torch.cuda.stream(streams[k]):
            x, w = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
            y = plstm.layer_norm(x, w)
            out = (y.detach(), *torch.autograd.grad(y, (x, w), dy))
        streams[k].synchronize()
        return out

    torch.cuda.synchronize()
    want, wrong = [call(k) for k in range(len(shapes))], []

    def work(k):
        try:
            for _ in range(40):
                if not all(torch.equal(a, b) for a, b in zip(call(k), want[k])):
                    wrong.append((shapes[k], "other bits"))
        except Exception as e:
            wrong.append((shapes[k], repr(e)))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(shapes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_regressor_with_lengths_is_the_rows_one_by_one(cuda_device):
    """Outputs within a row's length and its final states are those of the row alone; what stands past it, NaN
    included, counts nowhere."""
    torch.manual_seed(0)
    m = plstm.GatedScanRegressor(5, 64, 24, 3).to(cuda_device).eval()
    x, lens = _randn(4, 50, 5, dtype=F32, dev=cuda_device), [50, 1, 23, 0]
    for b, n in enumerate(lens):
        x[b, n:] = float("nan")
    with torch.no_grad():
        out, state = m(x, lengths=torch.tensor(lens))
        for b, n in enumerate(lens):
            alone, alone_state = m(x[b:b + 1, :n])
            # f32 GEMMs of another shape round differently: sums of 64 products.
            torch.testing.assert_close(out[b:b + 1, :n], alone, atol=2e-4, rtol=1e-3)
            for got, want in zip(state, alone_state):
                torch.testing.assert_close(got[b:b + 1], want, atol=2e-4, rtol=1e-3)
