"""Training and streaming operators over the C ABI, differentiable through autograd.

* ``gated_scan`` / ``gated_scan_step``: the recurrence of an LSTM layer whose gates do not
  look back, over a whole sequence (time is scanned in parallel) or one step of a stream.
* ``layer_norm``: over the last axis, up to 16384 wide.
* ``dropout``: from a counter-based generator, so the mask is never stored.
* ``dropout_add_layer_norm``: the residual step z = residual + dropout(x), y = layer_norm(z).

Inputs are CUDA tensors in f32, f16 or bf16; there is no CPU path.  Work is enqueued on the
current stream of the inputs' device.  The scan and the norms read strided batches, time
steps and rows in place; only a last axis that is not contiguous is copied first.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .core import _DTYPES, _ptr, _require_cuda, _stream

_byref = ctypes.byref
_MASK64 = (1 << 64) - 1


def _cuda_float(t: torch.Tensor, name: str) -> torch.Tensor:
    """`t` with a contiguous last axis; refuses what the kernels have no type for."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this path has no CPU implementation)")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} has dtype {t.dtype}; use float32, float16 or bfloat16")
    return t if t.dim() == 0 or t.stride(-1) == 1 else t.contiguous()


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- gated scan ------------------------------------------------------------------------------
def _scan_desc(gates: torch.Tensor, seq_major: bool) -> _lib.ScanDesc:
    b, t = (1, 0) if seq_major else (0, 1)
    return _lib.ScanDesc(gates.shape[b], gates.shape[t], gates.shape[2] // 4, _DTYPES[gates.dtype],
                         gates.device.index, 0, gates.stride(b), gates.stride(t), 0, 0, 0, 0)


def _scan_strides(d: _lib.ScanDesc, t: torch.Tensor, seq_major: bool, which: str) -> None:
    b, s = (t.stride(1), t.stride(0)) if seq_major else (t.stride(0), t.stride(1))
    setattr(d, which + "_batch_stride", b)
    setattr(d, which + "_time_stride", s)


def _scan_forward(gates, c0, lengths, seq_major, keep, c_n=None):
    lib = _lib.load()
    dev = gates.device
    d = _scan_desc(gates, seq_major)
    h = torch.empty(gates.shape[0], gates.shape[1], d.hidden, dtype=gates.dtype, device=dev)
    _scan_strides(d, h, seq_major, "h")
    if c_n is None:
        c_n = torch.empty(d.batch, d.hidden, dtype=torch.float32, device=dev)
    ckpt = None
    if keep:
        nbytes = ctypes.c_size_t(0)
        _lib.check(lib.plstm_gated_scan_checkpoint_size(_byref(d), _byref(nbytes)))
        ckpt = torch.empty(nbytes.value // 4, dtype=torch.float32, device=dev)
    _lib.check(lib.plstm_gated_scan_forward(_byref(d), _ptr(gates), _ptr(lengths), _ptr(c0), _ptr(h), _ptr(c_n),
                                            _ptr(ckpt), _stream(dev)))
    return h, c_n, ckpt


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gates, c0, lengths, seq_major):
        h, c_n, ckpt = _scan_forward(gates, c0, lengths, seq_major, True)
        ctx.save_for_backward(gates, lengths, ckpt)
        ctx.seq_major = seq_major
        ctx.set_materialize_grads(False)
        return h, c_n

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dc_n):
        gates, lengths, ckpt = ctx.saved_tensors
        d = _scan_desc(gates, ctx.seq_major)
        if dh is not None:
            dh = dh if dh.stride(2) == 1 else dh.contiguous()
            _scan_strides(d, dh, ctx.seq_major, "h")
        if dc_n is not None:
            dc_n = dc_n.contiguous()
        dgates = torch.empty(gates.shape, dtype=gates.dtype, device=gates.device)
        _scan_strides(d, dgates, ctx.seq_major, "dgates")
        dc0 = torch.empty(d.batch, d.hidden, dtype=torch.float32, device=gates.device) if ctx.needs_input_grad[1] \
            else None
        _lib.check(_lib.load().plstm_gated_scan_backward(
            _byref(d), _ptr(gates), _ptr(lengths), _ptr(ckpt), _ptr(dh), _ptr(dc_n), _ptr(dgates), _ptr(dc0),
            _stream(gates.device)))
        return dgates, dc0, None, None


def gated_scan(gates: torch.Tensor, c0: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, *,
               seq_major: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gate projections -> (h, c_n) of an LSTM layer whose gates do not look back.

    gates [B,T,4H] (or [T,B,4H] with seq_major=True) holds the pre-activations in nn.LSTM's gate
    order i, f, g, o:  c_t = sigmoid(f) c_{t-1} + sigmoid(i) tanh(g),  h_t = sigmoid(o) tanh(c_t).
    c0 [B,H] f32 (default zeros); lengths [B]: the state stands still from a row's length on, h is
    zero there, and neither the gates nor their gradient count.  Returns h in the gates' type and
    layout and c_n [B,H] f32.  Differentiable in gates and c0.
    """
    gates = _cuda_float(gates, "gates")
    if gates.dim() != 3 or gates.shape[2] == 0 or gates.shape[2] % 4:
        raise ValueError(f"gates must be [B, T, 4H] with H >= 1, got {tuple(gates.shape)}")
    B, H = gates.shape[1 if seq_major else 0], gates.shape[2] // 4
    if c0 is not None:
        c0 = _require_cuda(c0, "c0", gates.device, torch.float32)
        if c0.shape != (B, H):
            raise ValueError(f"c0 must be [{B}, {H}], got {tuple(c0.shape)}")
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.is_floating_point() or lengths.shape != (B,):
            raise ValueError(f"lengths must be an integer tensor [{B}]")
        lengths = lengths.to(device=gates.device, dtype=torch.int32).contiguous()
    if _wants_grad(gates, c0):
        return _GatedScan.apply(gates, c0, lengths, seq_major)
    h, c_n, _ = _scan_forward(gates, c0, lengths, seq_major, False)
    return h, c_n


def gated_scan_step(gates: torch.Tensor, c: torch.Tensor, *,
                    out_c: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One time step of ``gated_scan`` for a batch of streams: gates [B,4H], state c [B,H] f32 -> (h, c_new).

    out_c (f32 [B,H], contiguous) receives the new state; out_c=c updates the state in place.
    """
    gates = _cuda_float(gates, "gates")
    if gates.dim() != 2:
        raise ValueError(f"gates must be [B, 4H], got {tuple(gates.shape)}")
    if out_c is None:
        h, c_n = gated_scan(gates[:, None], c)
        return h[:, 0], c_n
    if _wants_grad(gates, c):
        raise ValueError("gated_scan_step with out_c is not differentiable; call it without out_c or under no_grad")
    B, H = gates.shape[0], gates.shape[1] // 4
    if H < 1 or gates.shape[1] % 4:
        raise ValueError(f"gates must be [B, 4H] with H >= 1, got {tuple(gates.shape)}")
    c = _require_cuda(c, "c", gates.device, torch.float32)
    _require_cuda(out_c, "out_c", gates.device, torch.float32)
    if c.shape != (B, H) or out_c.shape != (B, H) or not out_c.is_contiguous():
        raise ValueError(f"c and out_c must be [{B}, {H}], out_c contiguous")
    h, c_n, _ = _scan_forward(gates[:, None], c, None, False, False, out_c)
    return h[:, 0], c_n


# ---- dropout --------------------------------------------------------------------------------
def _drop_desc(p: float, seed: Union[int, torch.Tensor], offset: int, device: torch.device) -> _lib.DropoutDesc:
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if not 0 <= offset <= _MASK64:
        raise ValueError("offset must be in [0, 2^64)")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"a tensor seed must be one int64 on {device}")
        return _lib.DropoutDesc(p, 0, offset, seed.data_ptr())
    if not 0 <= seed <= _MASK64:
        raise ValueError("seed must be in [0, 2^64)")
    return _lib.DropoutDesc(p, seed, offset, None)


def _dropout(x, p, seed, offset, residual, dtype):
    y = torch.empty(x.shape, dtype=dtype, device=x.device)
    _lib.check(_lib.load().plstm_dropout(_byref(_drop_desc(p, seed, offset, x.device)), x.numel(), _ptr(x),
                                         _DTYPES[x.dtype], _ptr(residual), _ptr(y), _DTYPES[dtype], x.device.index,
                                         _stream(x.device)))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.args = (p, None if isinstance(seed, torch.Tensor) else seed, offset, x.dtype)
        ctx.save_for_backward(seed if isinstance(seed, torch.Tensor) else None)
        return _dropout(x, p, seed, offset, residual, x.dtype if residual is None else residual.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed, offset, dtype = ctx.args
        dx = None
        if ctx.needs_input_grad[0]:
            dx = _dropout(dy.contiguous(), p, ctx.saved_tensors[0] if seed is None else seed, offset, None, dtype)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def _check_residual(residual: torch.Tensor, x: torch.Tensor) -> None:
    if residual.device != x.device or residual.shape != x.shape:
        raise ValueError(f"residual must be {tuple(x.shape)} on {x.device}, got {tuple(residual.shape)} on "
                         f"{residual.device}")
    if residual.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"residual must be {x.dtype} or float32, got {residual.dtype}")


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], offset: int = 0, *,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dropout(x), or residual + dropout(x), with the mask a function of (seed, offset, element).

    Element e of the flattened x is kept where word e % 4 of Philox4x32-10 at counter
    (e // 4, offset) under key `seed` is >= floor(p * 2^32), and scaled by 1 / (1 - p); a dropped
    element is zero whatever it holds.  Calls that must draw apart need another seed or offset.
    seed: an int, or one int64 on the GPU (read by the kernel, so a captured graph draws anew
    when the tensor is advanced before the next replay).  The residual (x's type or f32) sets the
    result's type.  Differentiable in x and residual.
    """
    x = _cuda_float(x, "x").contiguous()
    if residual is not None:
        residual = _cuda_float(residual, "residual").contiguous()
        _check_residual(residual, x)
    if _wants_grad(x, residual):
        return _Dropout.apply(x, residual, p, seed, offset)
    return _dropout(x, p, seed, offset, residual, x.dtype if residual is None else residual.dtype)


# ---- layer norm -------------------------------------------------------------------------------
def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as [rows, cols] with contiguous columns (a view wherever the strides allow one)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _norm_desc(x, z_dtype, w_dtype, eps) -> _lib.NormDesc:
    return _lib.NormDesc(x.shape[0], x.shape[1], _DTYPES[x.dtype], _DTYPES[z_dtype], _DTYPES[w_dtype],
                         x.device.index, eps, x.stride(0), 0, 0, 0)


def _norm_forward(x, residual, weight, bias, eps, drop, keep):
    """x, residual [rows, cols] -> (y, z or None, stats or None)."""
    lib = _lib.load()
    dev = x.device
    w_dtype = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
    d = _norm_desc(x, x.dtype if residual is None else residual.dtype, w_dtype, eps)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    z = None
    if residual is not None:
        z = torch.empty(x.shape, dtype=residual.dtype, device=dev)
        d.residual_stride = residual.stride(0)
    stats = torch.empty(2, x.shape[0], dtype=torch.float32, device=dev) if keep else None
    _lib.check(lib.plstm_layer_norm_forward(_byref(d), None if drop is None else _byref(drop), _ptr(x),
                                            _ptr(residual), _ptr(weight), _ptr(bias), _ptr(z), _ptr(y), _ptr(stats),
                                            _stream(dev)))
    return y, z, stats


def _norm_backward(v, weight, stats, dy, dz, eps, drop, x_dtype, w_dtype, need_dx, need_dres, need_dw, need_db):
    """Gradients of (x, residual, weight, bias); drop is None for the plain norm."""
    lib = _lib.load()
    dev = v.device
    fused = drop is not None
    d = _lib.NormDesc(v.shape[0], v.shape[1], _DTYPES[x_dtype], _DTYPES[v.dtype], _DTYPES[w_dtype], dev.index, eps,
                      v.stride(0), 0, dy.stride(0), 0 if dz is None else dz.stride(0))
    dx = torch.empty(v.shape, dtype=x_dtype, device=dev) if need_dx else None
    dres = torch.empty(v.shape, dtype=v.dtype, device=dev) if need_dres else None
    dw = torch.empty(v.shape[1], dtype=w_dtype, device=dev) if need_dw else None
    db = torch.empty(v.shape[1], dtype=w_dtype, device=dev) if need_db else None
    ws, nbytes = None, ctypes.c_size_t(0)
    if need_dw or need_db:
        _lib.check(lib.plstm_layer_norm_backward_workspace_size(_byref(d), _byref(nbytes)))
        ws = torch.empty(max(nbytes.value, 16), dtype=torch.uint8, device=dev)
    _lib.check(lib.plstm_layer_norm_backward(_byref(d), _byref(drop) if fused else None, 1 if fused else 0, _ptr(dy),
                                             _ptr(dz), _ptr(v), _ptr(weight), _ptr(stats), _ptr(dx), _ptr(dres),
                                             _ptr(dw), _ptr(db), _ptr(ws), nbytes.value, _stream(dev)))
    return dx, dres, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows = _rows(x)
        y, _, stats = _norm_forward(rows, None, weight, bias, eps, None, True)
        ctx.save_for_backward(rows, weight, stats)
        ctx.eps, ctx.w_dtype = eps, x.dtype if weight is None and bias is None else \
            (bias if weight is None else weight).dtype
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, _, dw, db = _norm_backward(x, weight, stats, _rows(dy), None, ctx.eps, None, x.dtype, ctx.w_dtype,
                                       need[0], False, need[1], need[2])
        return None if dx is None else dx.view(dy.shape), dw, db, None


class _DropoutAddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, p, seed, offset, eps):
        y, z, stats = _norm_forward(_rows(x), _rows(residual), weight, bias, eps,
                                    _drop_desc(p, seed, offset, x.device), True)
        ctx.save_for_backward(z, weight, stats, seed if isinstance(seed, torch.Tensor) else None)
        ctx.args = (p, None if isinstance(seed, torch.Tensor) else seed, offset, eps)
        ctx.x_dtype = x.dtype
        ctx.w_dtype = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
        ctx.set_materialize_grads(False)
        return y.view(x.shape), z.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dz):
        z, weight, stats, seed_t = ctx.saved_tensors
        p, seed, offset, eps = ctx.args
        if dy is None and dz is None:
            return (None,) * 8
        shape = (dz if dy is None else dy).shape
        drop = _drop_desc(p, seed_t if seed is None else seed, offset, z.device)
        dy = torch.zeros((1, z.shape[1]), dtype=ctx.x_dtype, device=z.device).expand(z.shape) if dy is None \
            else _rows(dy)
        need = ctx.needs_input_grad
        dx, dres, dw, db = _norm_backward(z, weight, stats, dy, None if dz is None else _rows(dz), eps, drop,
                                          ctx.x_dtype, ctx.w_dtype, need[0], need[1], need[2], need[3])
        return (None if dx is None else dx.view(shape), None if dres is None else dres.view(shape), dw, db, None,
                None, None, None)


def _check_norm(x: torch.Tensor, weight, bias):
    if x.dim() == 0 or not 1 <= x.shape[-1] <= _lib.NORM_MAX_COLS:
        raise ValueError(f"the last axis must be 1 to {_lib.NORM_MAX_COLS} wide, got shape {tuple(x.shape)}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.device != x.device or t.shape != x.shape[-1:]:
            raise ValueError(f"{name} must be [{x.shape[-1]}] on {x.device}, got {tuple(t.shape)} on {t.device}")
        if t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must be {x.dtype} or float32, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one dtype")
    return (None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous())


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis, in x's type.

    weight and bias: x's type or f32.  Statistics, and the sums behind the weights' gradients,
    are f32.  Differentiable in x, weight and bias.
    """
    x = _cuda_float(x, "x")
    weight, bias = _check_norm(x, weight, bias)
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(_rows(x), None, weight, bias, eps, None, False)[0].view(x.shape)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                           bias: Optional[torch.Tensor] = None, p: float = 0.0,
                           seed: Union[int, torch.Tensor] = 0, offset: int = 0, *,
                           eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """The residual step in one pass: z = residual + dropout(x), y = layer_norm(z) -> (y, z).

    Bit for bit dropout(x, p, seed, offset, residual=residual) followed by the norm of that
    stored z.  The residual stream may be f32 under a 16-bit x; z has its type, y has x's.
    Differentiable in x, residual, weight and bias.
    """
    x = _cuda_float(x, "x")
    residual = _cuda_float(residual, "residual")
    _check_residual(residual, x)
    weight, bias = _check_norm(x, weight, bias)
    if _wants_grad(x, residual, weight, bias):
        return _DropoutAddLayerNorm.apply(x, residual, weight, bias, p, seed, offset, eps)
    y, z, _ = _norm_forward(_rows(x), _rows(residual), weight, bias, eps, _drop_desc(p, seed, offset, x.device),
                            False)
    return y.view(x.shape), z.view(x.shape)
