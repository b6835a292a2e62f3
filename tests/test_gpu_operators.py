"""The training and streaming operators on the GPU against their 64-bit forms, within elementwise
bounds that follow from f32 arithmetic and one rounding (operator_forms)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import operator_forms as forms
from operator_forms import assert_within, f64
import persistent_lstm_hip_b200 as plstm

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ZERO = torch.zeros((), dtype=torch.float64)


def _randn(*shape, dtype, dev, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 31 * len(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dev, dtype)


def _gates(B, T, H, dtype, dev, seed=0):
    g = torch.randn(B, T, 4 * H, generator=torch.Generator().manual_seed(seed))
    g[..., H:2 * H] += torch.linspace(-1, 5, H)
    return g.to(dev, dtype)


# ---- gated scan -----------------------------------------------------------------------------
def _check_scan(gates, c0, lengths, dh, dc_n, seq_major=False):
    """Runs forward and backward and compares both with the 64-bit form."""
    g = gates.detach().requires_grad_(True)
    c = None if c0 is None else c0.detach().requires_grad_(True)
    h, c_n = plstm.gated_scan(g, c, lengths, seq_major=seq_major)
    with torch.no_grad():
        h2, c2 = plstm.gated_scan(gates, c0, lengths, seq_major=seq_major)
    assert torch.equal(h, h2) and torch.equal(c_n, c2)
    grads = torch.autograd.grad((h, c_n), (g,) if c is None else (g, c), (dh, dc_n))
    flip = (lambda t: t.transpose(0, 1)) if seq_major else (lambda t: t)
    s = forms.scan_forward(f64(flip(gates)), f64(c0), None if lengths is None else lengths.cpu().long())
    r = forms.scan_backward(s, f64(flip(dh)), f64(dc_n))
    assert_within(flip(h), s["h"], s["h_err"], "h")
    assert_within(c_n, s["c_n"], s["c_n_err"], "c_n")
    assert_within(flip(grads[0]), r["dgates"], r["dgates_err"], "dgates")
    if c is not None:
        assert_within(grads[1], r["dc0"], r["dc0_err"], "dc0")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,T,H", [
    (1, 1, 1), (2, 7, 3), (1, 8, 64), (3, 9, 33), (1, 64, 66), (2, 65, 31), (5, 200, 8), (1, 257, 130),
    (1, 1023, 64), (2, 2050, 34), (1, 5000, 64), (40, 33, 128), (300, 17, 6), (700, 40, 64),
])
def test_scan_sizes(cuda_device, dtype, B, T, H):
    d = cuda_device
    _check_scan(_gates(B, T, H, dtype, d), _randn(B, H, dtype=F32, dev=d), None, _randn(B, T, H, dtype=dtype, dev=d),
                _randn(B, H, dtype=F32, dev=d, seed=1))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H", [(6, 37, 5), (6, 300, 64), (6, 2500, 32), (400, 90, 64)])
def test_scan_lengths_with_garbage_behind_them(cuda_device, dtype, B, T, H):
    """Lengths 0, 1, T, out of range on both sides and odd ones; what stands past a length is NaN or
    infinite and must count nowhere."""
    d = cuda_device
    lens = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(3))
    lens[:6] = torch.tensor([0, 1, T, T + 100, -5, T // 2])
    gates, dh = _gates(B, T, H, dtype, d), _randn(B, T, H, dtype=dtype, dev=d)
    dead = torch.arange(T)[None, :] >= lens[:, None]
    gates[dead.to(d)] = float("nan")
    gates[(dead & (torch.arange(T) % 3 == 0)).to(d)] = float("inf")
    dh[dead.to(d)] = float("nan")
    _check_scan(gates, _randn(B, H, dtype=F32, dev=d), lens.to(d, torch.int32), dh,
                _randn(B, H, dtype=F32, dev=d, seed=1))


def test_scan_without_initial_state_and_with_one_gradient_only(cuda_device):
    d, (B, T, H) = cuda_device, (3, 70, 40)
    gates, dh, dc_n = _gates(B, T, H, F32, d), _randn(B, T, H, dtype=F32, dev=d), _randn(B, H, dtype=F32, dev=d)
    _check_scan(gates, None, None, dh, dc_n)
    s = forms.scan_forward(f64(gates))
    for h_grad, c_grad in ((dh, None), (None, dc_n)):
        g = gates.clone().requires_grad_(True)
        h, c_n = plstm.gated_scan(g)
        (got,) = torch.autograd.grad([t for t, v in ((h, h_grad), (c_n, c_grad)) if v is not None], g,
                                     [v for v in (h_grad, c_grad) if v is not None])
        r = forms.scan_backward(s, f64(h_grad), f64(c_grad))
        assert_within(got, r["dgates"], r["dgates_err"], "dgates")


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("odd", [0, 1])
def test_scan_strided_inputs(cuda_device, dtype, odd):
    """Gates and dh as slices of wider tensors (odd offsets break the pair alignment), a last axis
    that is not contiguous, and a broadcast gradient."""
    d, (B, T, H) = cuda_device, (4, 50, 22)
    wide = _randn(B, T, 4 * H + 10 + odd, dtype=dtype, dev=d)
    gates = wide[..., odd:odd + 4 * H]
    dh = _randn(B, T, H + 6 + odd, dtype=dtype, dev=d)[..., odd:odd + H]
    c0, dc_n = _randn(B, H, dtype=F32, dev=d), _randn(B, H, dtype=F32, dev=d, seed=1)
    assert not gates.is_contiguous() and not dh.is_contiguous()
    _check_scan(gates, c0, None, dh, dc_n)
    _check_scan(gates.transpose(1, 2).contiguous().transpose(1, 2), c0, None, dh[:1, :1].expand(B, T, H), dc_n)
    _check_scan(gates[::2, ::3], c0[::2], None, dh[::2, ::3], dc_n[::2])
    _check_scan(gates, c0, None, dh[:1, :1, :1].expand(B, T, H), dc_n)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_seq_major(cuda_device, dtype):
    d, (B, T, H) = cuda_device, (5, 130, 24)
    gates = _gates(B, T, H, dtype, d).transpose(0, 1).contiguous()
    lens = torch.tensor([0, 1, 130, 64, 77], device=d)
    _check_scan(gates, _randn(B, H, dtype=F32, dev=d), lens, _randn(T, B, H, dtype=dtype, dev=d),
                _randn(B, H, dtype=F32, dev=d, seed=1), seq_major=True)


def test_scan_extreme_gates(cuda_device):
    """Saturated and infinite gates: sigmoid and tanh reach their limits, nothing overflows."""
    d, (B, T, H) = cuda_device, (2, 40, 16)
    inf = float("inf")
    for dtype in (F32, F16, BF16):
        gates = _gates(B, T, H, dtype, d)
        vals = torch.tensor([inf, -inf, 200.0, -200.0, 60.0, -60.0, 1e4, -1e4], device=d, dtype=dtype)
        gates.view(-1)[::5] = vals[torch.arange(gates.numel() // 5 + (gates.numel() % 5 > 0), device=d) % 8]
        _check_scan(gates, _randn(B, H, dtype=F32, dev=d), None, _randn(B, T, H, dtype=dtype, dev=d),
                    _randn(B, H, dtype=F32, dev=d, seed=1))


def test_scan_nan_stays_in_its_channel(cuda_device):
    d, (B, T, H) = cuda_device, (2, 100, 32)
    for dtype in (F32, BF16):
        gates = _gates(B, T, H, dtype, d)
        clean, _ = plstm.gated_scan(gates)
        gates[1, 40, H + 7] = float("nan")  # a forget gate
        h, c_n = plstm.gated_scan(gates)
        assert torch.isnan(h[1, 40:, 7]).all() and torch.isnan(c_n[1, 7])
        h[1, 40:, 7] = clean[1, 40:, 7]
        assert torch.equal(h, clean)


def test_scan_small_gates_keep_their_relative_precision(cuda_device):
    """tanh of small candidates: the state is right relatively, not only to 2^-24 of 1."""
    d, (B, T, H) = cuda_device, (2, 30, 16)
    for dtype in (F32, BF16):
        gates = _gates(B, T, H, dtype, d)
        gates[..., 2 * H:3 * H] *= 1e-3
        _check_scan(gates, None, None, _randn(B, T, H, dtype=dtype, dev=d), _randn(B, H, dtype=F32, dev=d))


def test_scan_empty(cuda_device):
    d = cuda_device
    c0 = _randn(3, 5, dtype=F32, dev=d)
    h, c_n = plstm.gated_scan(torch.empty(3, 0, 20, device=d), c0)
    assert h.shape == (3, 0, 5) and torch.equal(c_n, c0)
    h, c_n = plstm.gated_scan(torch.empty(0, 4, 20, device=d))
    assert h.shape == (0, 4, 5) and c_n.shape == (0, 5)
    g = torch.empty(3, 0, 20, device=d, requires_grad=True)
    c = c0.clone().requires_grad_(True)
    h, c_n = plstm.gated_scan(g, c)
    dg, dc = torch.autograd.grad(c_n, (g, c), torch.ones_like(c_n))
    assert dg.shape == g.shape and torch.equal(dc, torch.ones_like(c))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,H", [(1, 1), (1, 64), (3, 17), (16, 512), (1000, 96)])
def test_scan_step_streams(cuda_device, dtype, B, H):
    """Steps in place equal the scan over the same gates, state and outputs."""
    d, T = cuda_device, 11
    gates, c = _gates(B, T, H, dtype, d), _randn(B, H, dtype=F32, dev=d)
    s = forms.scan_forward(f64(gates), f64(c))
    new = c.clone()
    for t in range(T):
        before = new.clone()
        h_o, c_o = plstm.gated_scan_step(gates[:, t], before)
        assert torch.equal(before, new)
        h, out = plstm.gated_scan_step(gates[:, t], new, out_c=new)
        assert out is new and torch.equal(h, h_o) and torch.equal(new, c_o)
        assert_within(h, s["h"][:, t], s["h_err"][:, t], f"h at {t}")
    assert_within(new, s["c_n"], s["c_n_err"], "c_n")


def test_scan_is_the_hidden_update_without_recurrent_weights(cuda_device):
    from persistent_lstm_hip_b200 import adaptive_ext
    d, (B, T, H) = cuda_device, (3, 60, 20)
    gates = _gates(B, T, H, F32, d)
    h = torch.empty(B, H, device=d)
    c = torch.empty(B, H, device=d)
    out = torch.empty(B, T, H, device=d)
    adaptive_ext._hidden_update("test", gates, torch.zeros(4 * H, H, device=d), 0, torch.zeros(4 * H, device=d), h, c,
                                out, True)
    h2, c2 = plstm.gated_scan(gates)
    s = forms.scan_forward(f64(gates))
    assert ((h2 - out).abs().cpu() <= 2 * s["h_err"] + 1e-6).all()
    assert ((c2 - c).abs().cpu() <= 2 * s["c_n_err"] + 1e-6).all()


def test_scan_past_32_bit_offsets(cuda_device):
    """4 * T * H passes 2^32 elements: the two halves run apart must give the same."""
    d, (T, H) = cuda_device, (2_200_003, 512)
    gates = torch.empty(1, T, 4 * H, device=d, dtype=BF16)
    for part in gates.split(100_000, 1):
        part.normal_()
    assert gates.numel() > 1 << 32
    cut = 1_100_000
    h, c_n = plstm.gated_scan(gates)
    h1, c1 = plstm.gated_scan(gates[:, :cut])
    h2, c2 = plstm.gated_scan(gates[:, cut:], c1)
    # Segments fold in another order after the cut; errors fade with the forget gates, so every
    # value is within EPS / (1 - f) of its own size: 1e-3 covers f up to 0.998.
    assert torch.equal(h[:, :1000], h1[:, :1000])
    for a, b in ((h[:, :cut], h1), (h[:, cut:], h2)):
        for x, y in zip(a.split(200_000, 1), b.split(200_000, 1)):
            assert (x.float() - y.float()).abs().max() <= 2.0 ** -7
    assert (c_n - c2).abs().max() <= 1e-3
    s = forms.scan_forward(f64(gates[:, -300:]), f64(plstm.gated_scan(gates[:, :-300])[1]))
    assert_within(h[:, -300:], s["h"], s["h_err"] + 1e-3, "tail")
    del h1, h2
    g = gates[:, -cut:].requires_grad_(True)  # a view whose gradient alone passes 2^31 elements
    hg, _ = plstm.gated_scan(g)
    (dg,) = torch.autograd.grad(hg, g, torch.ones((), device=d, dtype=BF16).expand_as(hg))
    r = forms.scan_backward(forms.scan_forward(f64(gates[:, -300:].detach()), f64(plstm.gated_scan(
        gates[:, -cut:-300].detach())[1])), torch.ones(1, 300, H, dtype=torch.float64))
    assert_within(dg[:, -300:], r["dgates"], r["dgates_err"] + 1e-3, "tail of dgates")


def test_scan_gradient_against_differences_of_the_kernel(cuda_device):
    """Central differences of the forward kernel along random directions.  With h = 1e-2 the
    third-order term is below 1e-4 of the sum of |grad v| and f32 rounding (1e-6 of |h dh| over
    2e-2) below 1e-4 of the sum of |h dh|."""
    d, (B, T, H) = cuda_device, (2, 150, 16)
    gates, c0, dh = _gates(B, T, H, F32, d), _randn(B, H, dtype=F32, dev=d), _randn(B, T, H, dtype=F32, dev=d)
    g, c = gates.clone().requires_grad_(True), c0.clone().requires_grad_(True)
    h, _ = plstm.gated_scan(g, c)
    dg, dc = torch.autograd.grad(h, (g, c), dh)
    for seed in range(3):
        v, u = _randn(B, T, 4 * H, dtype=F32, dev=d, seed=50 + seed), _randn(B, H, dtype=F32, dev=d, seed=60 + seed)
        f = lambda s: (plstm.gated_scan(gates + s * v, c0 + s * u)[0].double() * dh.double()).sum()
        got = (f(1e-2) - f(-1e-2)) / 2e-2
        want = (dg.double() * v).sum() + (dc.double() * u).sum()
        room = 1e-4 * ((dg * v).abs().double().sum() + (dc * u).abs().double().sum() + (h * dh).abs().double().sum())
        assert (got - want).abs() <= room, (got, want, room)


def test_scan_twice_gives_the_same_bits(cuda_device):
    d, (B, T, H) = cuda_device, (2, 9000, 64)
    gates, dh = _gates(B, T, H, BF16, d), _randn(B, T, H, dtype=BF16, dev=d)
    first = None
    for _ in range(5):
        g = gates.clone().requires_grad_(True)
        h, c_n = plstm.gated_scan(g)
        out = (h, c_n, *torch.autograd.grad(h, g, dh))
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(out, first))


def test_scan_on_another_stream_and_in_a_graph(cuda_device):
    d, (B, T, H) = cuda_device, (2, 300, 64)
    gates, c = _gates(B, T, H, BF16, d), torch.zeros(B, H, device=d)
    want, want_c = plstm.gated_scan(gates, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_c = plstm.gated_scan(gates, c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(got_c, want_c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, c_n = plstm.gated_scan(gates, c)
    gates.copy_(gates.flip(1))
    graph.replay()
    flipped, _ = plstm.gated_scan(gates, c)
    assert torch.equal(h, flipped)


def test_scan_refusals(cuda_device):
    d = cuda_device
    x = torch.zeros(2, 3, 8, device=d)
    for bad, kw, msg in ((x[0], {}, "4H"), (x[..., :6], {}, "4H"), (x.double(), {}, "float64"), (x.long(), {}, "int64"),
                         (x, dict(c0=torch.zeros(2, 3, device=d)), "c0"),
                         (x, dict(c0=torch.zeros(2, 2, device=d).half()), "c0"),
                         (x, dict(c0=torch.zeros(2, 2)), "c0"),
                         (x, dict(lengths=torch.zeros(3, device=d, dtype=torch.int32)), "lengths"),
                         (x, dict(lengths=torch.zeros(2, device=d)), "lengths")):
        with pytest.raises(ValueError, match=msg):
            plstm.gated_scan(bad, **kw)
    c = torch.zeros(2, 2, device=d)
    with pytest.raises(ValueError, match="differentiable"):
        plstm.gated_scan_step(x[:, 0].clone().requires_grad_(True), c, out_c=c)
    with pytest.raises(ValueError, match="contiguous"):
        plstm.gated_scan_step(x[:, 0], c, out_c=torch.zeros(2, 2, device=d).t())


# ---- layer norm -----------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (3, 2), (5, 7), (1, 8), (70, 31), (33, 64), (9, 127), (130, 128), (40, 255), (17, 256),
               (600, 512), (3, 515), (30, 1000), (1000, 1024), (7, 1025), (5, 4096), (6, 4097), (2, 8192), (3, 16383),
               (20, 16384)]


def _check_norm(x, w, b, dy, eps=1e-5):
    args = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    it = iter(args)
    xg, wg, bg = next(it), next(it) if w is not None else None, next(it) if b is not None else None
    y = plstm.layer_norm(xg, wg, bg, eps)
    with torch.no_grad():
        assert torch.equal(plstm.layer_norm(x, w, b, eps), y)
    assert y.dtype == x.dtype and y.shape == x.shape
    grads = iter(torch.autograd.grad(y, args, dy))
    N = x.shape[-1]
    s = forms.norm_forward(f64(x).reshape(-1, N), f64(w), f64(b), eps)
    r = forms.norm_backward(s, f64(dy).reshape(-1, N))
    assert_within(y.reshape(-1, N), s["y"], s["y_err"], "y")
    assert_within(next(grads).reshape(-1, N), r["dv"], r["dv_err"], "dx")
    if w is not None:
        assert_within(next(grads), r["dw"], r["dw_err"], "dweight")
    if b is not None:
        assert_within(next(grads), r["db"], r["db_err"], "dbias")


def _norm_inputs(M, N, dtype, wdtype, dev):
    return (_randn(M, N, dtype=dtype, dev=dev, scale=2.0) + 0.5, 1 + _randn(N, dtype=wdtype, dev=dev, scale=0.2),
            _randn(N, dtype=wdtype, dev=dev, seed=1, scale=0.2), _randn(M, N, dtype=dtype, dev=dev, seed=2))


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("M,N", NORM_SHAPES)
def test_norm_sizes(cuda_device, dtype, wdtype, M, N):
    _check_norm(*_norm_inputs(M, N, dtype, wdtype, cuda_device))


def test_norm_many_rows(cuda_device):
    _check_norm(*_norm_inputs(20011, 72, BF16, F32, cuda_device))
    _check_norm(*_norm_inputs(5003, 640, F32, F32, cuda_device))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_optional_weights(cuda_device, dtype):
    x, w, b, dy = _norm_inputs(12, 96, dtype, dtype, cuda_device)
    _check_norm(x, None, None, dy)
    _check_norm(x, w, None, dy)
    _check_norm(x, None, b, dy)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_norm_strided(cuda_device, dtype):
    """Row slices at aligned and odd offsets, three axes, a last axis that is not contiguous, every
    second row, broadcast rows, and broadcast gradients."""
    d, N = cuda_device, 64
    _, w, b, _ = _norm_inputs(1, N, dtype, dtype, d)
    wide = _randn(6, 5, N + 40, dtype=dtype, dev=d)
    dy = _randn(6, 5, N + 24, dtype=dtype, dev=d, seed=3)
    for k in (0, 8, 1, 3):
        _check_norm(wide[..., k:k + N], w, b, dy[..., k:k + N])
        _check_norm(wide[0, :, k:k + N], w, b, dy[0, :, k:k + N])
    _check_norm(wide[..., :N].transpose(0, 1), w, b, dy[..., :N].transpose(0, 1))
    _check_norm(wide[0, :, :N].t().contiguous().t(), w, b, dy[0, :, :N].t().contiguous().t())
    _check_norm(wide[::2, :, :N], w, b, dy[::2, :, :N])
    _check_norm(wide[:1, :1, :N].expand(6, 5, N), w, b, dy[..., :N])
    _check_norm(wide[..., :N], w, b, dy[:1, :1, :N].expand(6, 5, N))
    _check_norm(wide[..., :N], w, b, dy[:1, :1, :1].expand(6, 5, N))


def test_norm_far_from_zero_and_constant_rows(cuda_device):
    """A mean 1000 times the spread (two passes, no cancellation) and rows without any spread."""
    x, w, b, dy = _norm_inputs(9, 300, F32, F32, cuda_device)
    _check_norm(x + 1000.0, w, b, dy)
    const = torch.full_like(x, 2.0)
    y = plstm.layer_norm(const, w, b)
    assert torch.equal(y, b.expand_as(y))
    _check_norm(const, w, b, dy)


def test_norm_nan_and_inf_stay_in_their_row(cuda_device):
    for M, N in ((9, 48), (9, 2000)):
        x, w, b, _ = _norm_inputs(M, N, BF16, F32, cuda_device)
        clean = plstm.layer_norm(x, w, b)
        x[2, 3], x[5, 7] = float("nan"), float("inf")
        y = plstm.layer_norm(x, w, b)
        assert torch.isnan(y[2]).all() and torch.isnan(y[5]).all()
        y[2], y[5] = clean[2], clean[5]
        assert torch.equal(y, clean)


def test_norm_empty_and_refusals(cuda_device):
    d = cuda_device
    w = torch.ones(8, device=d, requires_grad=True)
    x = torch.empty(0, 8, device=d, requires_grad=True)
    y = plstm.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 8, device=d))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros(8, device=d))
    x = torch.zeros(2, 8, device=d)
    for bad in (lambda: plstm.layer_norm(x[:, :0]), lambda: plstm.layer_norm(torch.zeros(1, 16385, device=d)),
                lambda: plstm.layer_norm(x, torch.ones(7, device=d)), lambda: plstm.layer_norm(x.double()),
                lambda: plstm.layer_norm(x, torch.ones(8, device=d).half()), lambda: plstm.layer_norm(x, torch.ones(8)),
                lambda: plstm.layer_norm(x.half(), torch.ones(8, device=d).half(), torch.ones(8, device=d)),
                lambda: plstm.dropout_add_layer_norm(x, x[:1]), lambda: plstm.dropout_add_layer_norm(x, x.half()),
                lambda: plstm.dropout_add_layer_norm(x, x, p=1.5)):
        with pytest.raises(ValueError):
            bad()


# ---- dropout --------------------------------------------------------------------------------
def _exact_dropout(x, p, seed, offset, residual=None):
    """What the kernel must give bit for bit: the f32 product and sum, one rounding each."""
    keep = torch.zeros(x.shape, dtype=torch.bool) if p == 1 else \
        forms.keep_mask(np.arange(x.numel()), p, seed, offset).view(x.shape)
    y = torch.where(keep, x.cpu().float() * np.float32(1 / (1 - p) if p < 1 else 0), torch.zeros(()))
    if residual is not None:
        y = residual.cpu().float() + y
    return y.to(x.dtype if residual is None else residual.dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 31, 1000, 4097, 300001])
def test_dropout_is_the_published_generator(cuda_device, dtype, n):
    d, seed, offset = cuda_device, 0x9E3779B97F4A7C15, (1 << 40) + 5
    x = _randn(n, dtype=dtype, dev=d)
    dy = _randn(n, dtype=dtype, dev=d, seed=5)
    for p in (0.1, 0.5, 0.93):
        xg = x.clone().requires_grad_(True)
        y = plstm.dropout(xg, p, seed, offset)
        (dx,) = torch.autograd.grad(y, xg, dy)
        assert torch.equal(y.cpu(), _exact_dropout(x, p, seed, offset))
        assert torch.equal(dx.cpu(), _exact_dropout(dy, p, seed, offset))


@pytest.mark.parametrize("dtype,rdtype", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("n", [5, 64, 10007])
def test_dropout_with_a_residual(cuda_device, dtype, rdtype, n):
    d = cuda_device
    x, r = _randn(n, dtype=dtype, dev=d), _randn(n, dtype=rdtype, dev=d, seed=1)
    dy = _randn(n, dtype=rdtype, dev=d, seed=2)
    xg, rg = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
    y = plstm.dropout(xg, 0.3, 77, 3, residual=rg)
    assert torch.equal(y.cpu(), _exact_dropout(x, 0.3, 77, 3, r))
    dx, dr = torch.autograd.grad(y, (xg, rg), dy)
    assert torch.equal(dr, dy) and dx.dtype == dtype
    assert torch.equal(dx.cpu(), _exact_dropout(dy, 0.3, 77, 3).to(dtype))


def test_dropout_limits_and_dropped_garbage(cuda_device):
    d = cuda_device
    x = _randn(999, dtype=BF16, dev=d)
    assert torch.equal(plstm.dropout(x, 0.0, 1), x)
    x[::2], x[1::4] = float("nan"), float("inf")
    assert torch.equal(plstm.dropout(x, 1.0, 1), torch.zeros_like(x))
    y, keep = plstm.dropout(x, 0.4, 9).cpu(), forms.keep_mask(np.arange(999), 0.4, 9, 0)
    assert (y[~keep] == 0).all() and torch.equal(torch.isnan(y), torch.isnan(x.cpu()) & keep)
    assert plstm.dropout(x[:0], 0.5, 1).shape == (0,)


def test_dropout_unaligned_strided_and_shaped(cuda_device):
    d = cuda_device
    base = _randn(40, 50, dtype=F16, dev=d)
    for x in (base.view(-1)[1:778], base[:, 3:20], base.t(), base[::2], base[:1].expand(40, 50)):
        assert torch.equal(plstm.dropout(x, 0.25, 5, 6).cpu(), _exact_dropout(x.cpu().contiguous(), 0.25, 5, 6))


def test_dropout_seed_on_the_gpu(cuda_device):
    """A tensor seed equals the same int, a captured graph draws anew when it is advanced, and
    changing it between forward and backward is caught."""
    d = cuda_device
    x, seed = _randn(5000, dtype=F32, dev=d), torch.tensor([42], device=d)
    assert torch.equal(plstm.dropout(x, 0.5, seed, 1), plstm.dropout(x, 0.5, 42, 1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = plstm.dropout(x, 0.5, seed, 1)
    seed.fill_(43)
    graph.replay()
    assert torch.equal(y, plstm.dropout(x, 0.5, 43, 1))
    xg = x.clone().requires_grad_(True)
    out = plstm.dropout(xg, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_dropout_keeps_the_stated_share(cuda_device):
    """Of n = 2^22 elements p are dropped, within six standard deviations; other offsets draw apart."""
    n = 1 << 22
    x = torch.ones(n, device=cuda_device)
    for p in (0.05, 0.5, 0.9):
        a, b = (plstm.dropout(x, p, 11, o) != 0 for o in (0, 1))
        dev = (p * (1 - p) / n) ** 0.5
        assert abs(float((~a).double().mean()) - p) < 6 * dev
        assert abs(float((a & b).double().mean()) - (1 - p) ** 2) < 6 * ((1 - p) ** 2 / n) ** 0.5


def test_dropout_past_32_bit_elements(cuda_device):
    n = (1 << 32) + 4099
    x = torch.ones(n, device=cuda_device, dtype=F16)
    y = plstm.dropout(x, 0.5, 3, 4)
    at = np.concatenate([np.arange(64), np.arange((1 << 31) - 64, (1 << 31) + 64), np.arange((1 << 32) - 64, n)])
    keep = forms.keep_mask(at, 0.5, 3, 4)
    got = y[torch.from_numpy(at).to(cuda_device)].cpu()
    assert torch.equal(got, keep.to(F16) * 2)


def test_dropout_refusals(cuda_device):
    x = torch.zeros(8, device=cuda_device)
    for bad in (lambda: plstm.dropout(x, -0.1, 1), lambda: plstm.dropout(x, 0.5, -1), lambda: plstm.dropout(x, 0.5, 1 << 64),
                lambda: plstm.dropout(x, 0.5, 1, -2), lambda: plstm.dropout(x.long(), 0.5, 1),
                lambda: plstm.dropout(x, 0.5, torch.zeros(1, device=cuda_device)),
                lambda: plstm.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64)),
                lambda: plstm.dropout(x, 0.5, 1, residual=x[:4]), lambda: plstm.dropout(x, 0.5, 1, residual=x.half())):
        with pytest.raises(ValueError):
            bad()


# ---- dropout + residual + norm ------------------------------------------------------------------
FUSED_TYPES = [(F32, F32, F32), (F16, F16, F16), (F16, F32, F32), (BF16, BF16, F32), (BF16, F32, BF16)]


@pytest.mark.parametrize("dtype,rdtype,wdtype", FUSED_TYPES)
@pytest.mark.parametrize("M,N", [(1, 1), (3, 5), (40, 64), (9, 129), (300, 256), (7, 1000), (65, 1024), (3, 4097),
                                 (5, 8192), (3, 16384)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_fused_step(cuda_device, dtype, rdtype, wdtype, M, N, p):
    """Bit for bit the separate dropout and norm; gradients against the 64-bit form."""
    d, seed, offset, eps = cuda_device, 99, 7, 1e-5
    x, w, b, dy = _norm_inputs(M, N, dtype, wdtype, d)
    res, dz = _randn(M, N, dtype=rdtype, dev=d, seed=4), _randn(M, N, dtype=rdtype, dev=d, seed=5)
    args = [t.detach().requires_grad_(True) for t in (x, res, w, b)]
    y, z = plstm.dropout_add_layer_norm(*args, p, seed, offset, eps=eps)
    with torch.no_grad():
        y2, z2 = plstm.dropout_add_layer_norm(x, res, w, b, p, seed, offset, eps=eps)
    assert torch.equal(y, y2) and torch.equal(z, z2)
    assert torch.equal(z, plstm.dropout(x, p, seed, offset, residual=res))
    dx, dres, dw, db = torch.autograd.grad((y, z), args, (dy, dz))
    s = forms.norm_forward(f64(z), f64(w), f64(b), eps)
    r = forms.norm_backward(s, f64(dy), f64(dz))
    if rdtype == dtype:
        assert torch.equal(y, plstm.layer_norm(z, w, b, eps))
    assert_within(y, s["y"], s["y_err"], "y")
    assert_within(dres, r["dv"], r["dv_err"], "dresidual")
    assert_within(dx, forms.dropped(r["dv"], p, seed, offset), 2 * r["dv_err"] / (1 - p), "dx")
    assert_within(dw, r["dw"], r["dw_err"], "dweight")
    assert_within(db, r["db"], r["db_err"], "dbias")


def test_fused_step_partial_gradients_and_strides(cuda_device):
    d, (M, N) = cuda_device, (12, 48)
    x, w, b, dy = _norm_inputs(M, N, BF16, F32, d)
    wide = _randn(M, N + 16, dtype=BF16, dev=d, seed=8)
    res, dz = wide[:, 3:3 + N], _randn(M, N + 8, dtype=BF16, dev=d, seed=9)[:, 8:]
    for gy, gz, p in ((dy, None, 0.5), (None, dz, 0.5), (dy, dz, 1.0), (dy[:1].expand(M, N), dz[:1].expand(M, N), 0.2)):
        args = [t.detach().requires_grad_(True) for t in (x, res, w, b)]
        y, z = plstm.dropout_add_layer_norm(*args, p, 5, 1)
        outs = [(o, g) for o, g in ((y, gy), (z, gz)) if g is not None]
        grads = torch.autograd.grad([o for o, _ in outs], args, [g for _, g in outs], allow_unused=True)
        s = forms.norm_forward(f64(z), f64(w), f64(b), 1e-5)
        r = forms.norm_backward(s, torch.zeros(M, N, dtype=torch.float64) if gy is None else f64(gy), f64(gz))
        assert_within(grads[1], r["dv"], r["dv_err"], "dresidual")
        assert_within(grads[0], forms.dropped(r["dv"], p, 5, 1), 2 * r["dv_err"] / (1 - p) if p < 1 else
                      torch.zeros_like(r["dv_err"]), "dx")
        assert_within(grads[2], r["dw"], r["dw_err"], "dweight")


def test_fused_step_drops_garbage(cuda_device):
    d, (M, N) = cuda_device, (4, 64)
    x, w, b, _ = _norm_inputs(M, N, F16, F16, d)
    res = _randn(M, N, dtype=F16, dev=d, seed=4)
    keep = forms.keep_mask(np.arange(M * N), 0.5, 3, 0).view(M, N).to(d)
    want = plstm.dropout_add_layer_norm(x, res, w, b, 0.5, 3)
    got = plstm.dropout_add_layer_norm(x.masked_fill(~keep, float("nan")), res, w, b, 0.5, 3)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


# ---- the operators together -----------------------------------------------------------------------
def test_regressor_streams_what_it_computes_at_once(cuda_device):
    torch.manual_seed(0)
    m = plstm.GatedScanRegressor(5, 64, 24, 3).to(cuda_device).eval()
    x = _randn(4, 50, 5, dtype=F32, dev=cuda_device)
    with torch.no_grad():
        whole, state_n = m(x)
        state = m.init_state(4)
        steps = torch.stack([m.step(x[:, t], state) for t in range(50)], 1)
        half, mid = m(x[:, :20])
        rest, _ = m(x[:, 20:], state=mid)
    # f32 GEMMs of another shape round differently: 50 steps of sums of 64 products.
    torch.testing.assert_close(steps, whole, atol=2e-4, rtol=1e-3)
    torch.testing.assert_close(torch.cat([half, rest], 1), whole, atol=2e-4, rtol=1e-3)
    for a, b in zip(state, state_n):
        torch.testing.assert_close(a, b, atol=2e-4, rtol=1e-3)


def test_regressor_learns(cuda_device):
    """A stack in training mode learns a running mean of its inputs."""
    torch.manual_seed(0)
    m = plstm.GatedScanRegressor(4, 32, 1, 2, dropout=0.05).to(cuda_device).train()
    opt = torch.optim.Adam(m.parameters(), lr=1e-2)
    x = _randn(32, 40, 4, dtype=F32, dev=cuda_device)
    target = x.mean(-1).cumsum(1) / torch.arange(1, 41, device=cuda_device)
    losses = []
    for _ in range(60):
        opt.zero_grad()
        loss = ((m(x)[0][..., 0] - target) ** 2).mean()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    assert losses[-1] < 0.25 * losses[0], losses[::10]


def test_second_derivatives_are_refused(cuda_device):
    """Differentiating a gradient again is an error, never a silently wrong number; a recorded
    backward alone is not."""
    d = cuda_device
    x, g = _randn(4, 16, dtype=F32, dev=d).requires_grad_(True), _gates(2, 5, 4, F32, d).requires_grad_(True)
    for y, v in ((plstm.layer_norm(x), x), (plstm.dropout(x, 0.5, 1), x), (plstm.gated_scan(g)[0], g),
                 (plstm.dropout_add_layer_norm(x, x * 2)[0], x)):
        (d1,) = torch.autograd.grad((y * y).sum(), v, create_graph=True)
        assert torch.isfinite(d1).all()
        with pytest.raises(RuntimeError, match="once_differentiable|differentiated twice"):
            d1.sum().backward()
