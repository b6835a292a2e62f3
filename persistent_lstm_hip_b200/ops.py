"""Training and streaming operators over the C ABI, differentiable through autograd.

* ``gated_scan`` / ``gated_scan_step``: the recurrence of an LSTM layer whose gates do not
  look back, over a whole sequence (time is scanned in parallel) or one step of a stream.
* ``layer_norm``: over the last axis, up to 16384 wide.
* ``dropout``: from a counter-based generator, so the mask is never stored.
* ``dropout_add_layer_norm``: the residual step z = residual + dropout(x), y = layer_norm(z).

Inputs are CUDA tensors in f32, f16 or bf16; there is no CPU path.  Gradients are of the first
order and in reverse mode; forward mode, second derivatives and tracers are refused.  Work is enqueued on the
current stream of the inputs' device.  The scan and the norms read strided batches, time
steps and rows in place; only a last axis that is not contiguous is copied first.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _lib
from .core import _DTYPES, _require_cuda

_byref = ctypes.byref
_empty = torch.empty
_F32 = torch.float32
_MASK64 = (1 << 64) - 1
_MAX32 = (1 << 31) - 1
# The current stream's handle without building a torch.cuda.Stream: small calls are host-bound.
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    lambda index: torch.cuda.current_stream(index).cuda_stream
# What says that a tracer may be active, each some 0.1 us (get_proxy_mode alone takes 0.4 us): modes on the
# dispatcher's stack, and on the one above autograd.
_is_tracing = torch._C._is_tracing
_modes = torch._C._len_torch_dispatch_stack
_early_modes = torch._ops.mode_stack_state_for_pre_dispatch().count


def _refuse_transforms(*tensors) -> None:
    """Refuses what would lose a call without a word.  The kernels carry no forward-mode tangents, and a result
    without one reads as a derivative of zero.  A tracer (torch.jit.trace, make_fx) sees the allocations but not the
    launches, and what it records would return uninitialised memory."""
    if _is_tracing() or ((_modes() or _early_modes()) and get_proxy_mode() is not None):
        raise RuntimeError("this operator cannot be traced: its kernel is launched outside of torch's dispatcher")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("this operator has no forward-mode derivative")


def _first_order(backward):
    """once_differentiable, whose bookkeeping only a backward that is itself recorded needs."""
    recorded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        _refuse_transforms(*grads)
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


# autograd's apply() costs about 0.6 us an argument, so what is no tensor goes through it as one.
# What depends on shapes, strides and types alone (checks, descriptors, sizes) is worked out once for
# each combination and found again by it in these bounded caches.
_plan = functools.lru_cache(maxsize=512)


def _ptr(t: Optional[torch.Tensor]):
    """The address of a tensor's elements, NULL for None.  Tensors without memory of their own (DTensor and other
    wrappers) have no address, and NULL would read as an argument left out (where none may be, the library refuses
    it)."""
    if t is None:
        return None
    address = t.data_ptr()
    if not address and t.numel():
        raise ValueError(f"a {type(t).__name__} without memory of its own is not supported; pass a plain tensor")
    return address


def _cuda_float(t: torch.Tensor, name: str) -> torch.Tensor:
    """`t` with a contiguous last axis; refuses what the kernels have no type for."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this path has no CPU implementation)")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} has dtype {t.dtype}; use float32, float16 or bfloat16")
    return t if t.dim() == 0 or t.stride(-1) == 1 else t.contiguous()


# ---- gated scan ------------------------------------------------------------------------------
class _ScanPlan(NamedTuple):
    desc: object       # byref of the descriptor
    state: tuple       # [B, H]
    h: tuple           # shape of h
    checkpoints: int   # f32 elements
    keep: object       # the descriptor


@_plan
def _scan_plan(shape, strides, dtype, index, seq_major, dh_strides=None) -> _ScanPlan:
    if len(shape) != 3 or shape[2] == 0 or shape[2] % 4:
        raise ValueError(f"gates must be [B, T, 4H] with H >= 1, got {tuple(shape)}")
    if max(shape) > _MAX32:  # the descriptor's fields would wrap
        raise ValueError(f"gates must have axes below 2^31, got {tuple(shape)}")
    b, t = (1, 0) if seq_major else (0, 1)
    H = shape[2] // 4
    h = (shape[0], shape[1], H)
    h_strides = (shape[1] * H, H, 1) if dh_strides is None else dh_strides
    d_strides = (shape[1] * 4 * H, 4 * H, 1)
    d = _lib.ScanDesc(shape[b], shape[t], H, _DTYPES[dtype], index, 0, strides[b], strides[t], h_strides[b],
                      h_strides[t], d_strides[b], d_strides[t])
    nbytes = ctypes.c_size_t(0)
    _lib.check(_lib.load().plstm_gated_scan_checkpoint_size(_byref(d), _byref(nbytes)))
    return _ScanPlan(_byref(d), (shape[b], H), h, nbytes.value // 4, d)


@_plan
def _step_plan(shape, strides, dtype, index) -> _ScanPlan:
    """One step of [1, B, 4H]; h is allocated without the axis of one."""
    return _scan_plan((1, *shape), (0, *strides), dtype, index, True)


def _scan_forward(plan, gates, c0, lengths, keep):
    dev = gates.device
    h = _empty(plan.h, dtype=gates.dtype, device=dev)
    c_n = _empty(plan.state, dtype=_F32, device=dev)
    ckpt = _empty(plan.checkpoints, dtype=_F32, device=dev) if keep else None
    rc = _lib.load().plstm_gated_scan_forward(
        plan.desc, gates.data_ptr(), _ptr(lengths), _ptr(c0), h.data_ptr(), c_n.data_ptr(), _ptr(ckpt),
        _stream(dev.index))
    if rc:
        _lib.check(rc)
    return h, c_n, ckpt


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gates, c0, how):
        lengths, plan, seq_major = how
        h, c_n, ckpt = _scan_forward(plan, gates, c0, lengths, True)
        ctx.save_for_backward(gates, lengths, ckpt)
        ctx.seq_major = seq_major
        ctx.set_materialize_grads(False)
        return h, c_n

    @staticmethod
    @_first_order
    def backward(ctx, dh, dc_n):
        gates, lengths, ckpt = ctx.saved_tensors
        if dh is not None and dh.stride(2) != 1:
            dh = dh.contiguous()
        if dc_n is not None:
            dc_n = dc_n.contiguous()
        dev = gates.device
        plan = _scan_plan(gates.shape, gates.stride(), gates.dtype, dev.index, ctx.seq_major,
                          None if dh is None else dh.stride())
        dgates = _empty(gates.shape, dtype=gates.dtype, device=dev)
        dc0 = _empty(plan.state, dtype=_F32, device=dev) if ctx.needs_input_grad[1] else None
        rc = _lib.load().plstm_gated_scan_backward(
            plan.desc, gates.data_ptr(), _ptr(lengths), ckpt.data_ptr(), _ptr(dh), _ptr(dc_n), dgates.data_ptr(),
            _ptr(dc0), _stream(dev.index))
        if rc:
            _lib.check(rc)
        return dgates, dc0, None


def lengths32(lengths: torch.Tensor, batch: int, top: int, device: torch.device) -> torch.Tensor:
    """Checked lengths as the kernels take them: int32 on the device.  The kernels clamp to [0, top]; what int32
    cannot hold is clamped before it would wrap."""
    if not isinstance(lengths, torch.Tensor) or lengths.is_floating_point() or lengths.is_complex() or \
            lengths.shape != (batch,):
        raise ValueError(f"lengths must be an integer tensor [{batch}]")
    if lengths.dtype is torch.uint64:  # the upper half is negative as int64
        lengths = lengths.to(torch.int64)
        lengths = torch.where(lengths < 0, top, lengths)
    elif lengths.dtype is torch.uint32:
        lengths = lengths.to(torch.int64)
    if lengths.dtype is torch.int64:
        lengths = lengths.clamp(0, top)
    return lengths.to(device=device, dtype=torch.int32).contiguous()


def gated_scan(gates: torch.Tensor, c0: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, *,
               seq_major: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gate projections -> (h, c_n) of an LSTM layer whose gates do not look back.

    gates [B,T,4H] (or [T,B,4H] with seq_major=True) holds the pre-activations in nn.LSTM's gate
    order i, f, g, o:  c_t = sigmoid(f) c_{t-1} + sigmoid(i) tanh(g),  h_t = sigmoid(o) tanh(c_t).
    c0 [B,H] f32 (default zeros); lengths [B], clamped to [0, T]: the state stands still from a row's length on, h is
    zero there, and neither the gates nor their gradient count.  Returns h in the gates' type and
    layout and c_n [B,H] f32.  Differentiable in gates and c0.
    """
    _refuse_transforms(gates, c0)
    gates = _cuda_float(gates, "gates")
    plan = _scan_plan(gates.shape, gates.stride(), gates.dtype, gates.device.index, seq_major)
    if c0 is not None:
        c0 = _require_cuda(c0, "c0", gates.device, _F32)
        if c0.shape != plan.state:
            raise ValueError(f"c0 must be {list(plan.state)}, got {tuple(c0.shape)}")
    if lengths is not None:
        lengths = lengths32(lengths, plan.state[0], gates.shape[0 if seq_major else 1], gates.device)
    if torch.is_grad_enabled() and (gates.requires_grad or (c0 is not None and c0.requires_grad)):
        return _GatedScan.apply(gates, c0, (lengths, plan, seq_major))
    return _scan_forward(plan, gates, c0, lengths, False)[:2]


def gated_scan_step(gates: torch.Tensor, c: torch.Tensor, *,
                    out_c: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One time step of ``gated_scan`` for a batch of streams: gates [B,4H], state c [B,H] f32 -> (h, c_new).

    out_c (f32 [B,H], contiguous) receives the new state; out_c=c updates the state in place, any other
    must not overlap c.  Differentiable without out_c.
    """
    _refuse_transforms(gates, c, out_c)
    gates = _cuda_float(gates, "gates")
    if gates.dim() != 2:
        raise ValueError(f"gates must be [B, 4H], got {tuple(gates.shape)}")
    if torch.is_grad_enabled() and (gates.requires_grad or c.requires_grad or
                                    (out_c is not None and out_c.requires_grad)):
        if out_c is not None:
            raise ValueError("gated_scan_step with out_c is not differentiable; call it without out_c or under "
                             "no_grad")
        h, c_n = gated_scan(gates[:, None], c)
        return h[:, 0], c_n
    dev = gates.device
    plan = _step_plan(gates.shape, gates.stride(), gates.dtype, dev.index)
    c = _require_cuda(c, "c", dev, _F32)
    if c.shape != plan.state:
        raise ValueError(f"c must be {list(plan.state)}, got {tuple(c.shape)}")
    if out_c is None:
        out_c = _empty(plan.state, dtype=_F32, device=dev)
    else:
        _require_cuda(out_c, "out_c", dev, _F32)
        if out_c.shape != plan.state or not out_c.is_contiguous():
            raise ValueError(f"out_c must be {list(plan.state)} and contiguous")
        # The kernel writes behind autograd's back: a graph that saved this state has to notice.
        torch.autograd.graph.increment_version(out_c)
    h = _empty(plan.state, dtype=gates.dtype, device=dev)
    rc = _lib.load().plstm_gated_scan_forward(plan.desc, gates.data_ptr(), None, _ptr(c), h.data_ptr(),
                                              out_c.data_ptr(), None, _stream(dev.index))
    if rc:
        _lib.check(rc)
    return h, out_c


# ---- dropout --------------------------------------------------------------------------------
def _drop_desc(p: float, seed: Union[int, torch.Tensor], offset: int, device: torch.device) -> _lib.DropoutDesc:
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if not 0 <= offset <= _MASK64:
        raise ValueError("offset must be in [0, 2^64)")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"a tensor seed must be one int64 on {device}")
        return _lib.DropoutDesc(p, 0, offset, _ptr(seed))
    if not 0 <= seed <= _MASK64:
        raise ValueError("seed must be in [0, 2^64)")
    return _lib.DropoutDesc(p, seed, offset, None)


def _saved_drop(drop, seed):
    """The forward's descriptor for its backward.  A tensor seed is read where autograd holds it: saved-tensor
    hooks (checkpointing, offloading) keep a copy, and the forward's own tensor may be changed or freed by then."""
    return drop if seed is None else _lib.DropoutDesc(drop.p, 0, drop.offset, _ptr(seed))


def _dropout(x, drop, residual, dtype):
    dev = x.device
    y = _empty(x.shape, dtype=dtype, device=dev)
    rc = _lib.load().plstm_dropout(_byref(drop), x.numel(), x.data_ptr(), _DTYPES[x.dtype], _ptr(residual),
                                   y.data_ptr(), _DTYPES[dtype], dev.index, _stream(dev.index))
    if rc:
        _lib.check(rc)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, how):
        drop, seed = how
        ctx.args = (drop, x.dtype)
        # A tensor seed is kept with its version: changing it before the backward is an error.
        ctx.save_for_backward(seed)
        return _dropout(x, drop, residual, x.dtype if residual is None else residual.dtype)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        drop, dtype = ctx.args
        (seed,) = ctx.saved_tensors
        dx = _dropout(dy.contiguous(), _saved_drop(drop, seed), None, dtype) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None


def _check_residual(residual: torch.Tensor, x: torch.Tensor) -> None:
    if residual.device != x.device or residual.shape != x.shape:
        raise ValueError(f"residual must be {tuple(x.shape)} on {x.device}, got {tuple(residual.shape)} on "
                         f"{residual.device}")
    if residual.dtype is not x.dtype and residual.dtype is not _F32:
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
    _refuse_transforms(x, residual)
    x = _cuda_float(x, "x").contiguous()
    if residual is not None:
        residual = _cuda_float(residual, "residual").contiguous()
        _check_residual(residual, x)
    drop = _drop_desc(p, seed, offset, x.device)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, (drop, seed if isinstance(seed, torch.Tensor) else None))
    return _dropout(x, drop, residual, x.dtype if residual is None else residual.dtype)


# ---- layer norm -------------------------------------------------------------------------------
class _NormPlan(NamedTuple):
    desc: object      # byref of the descriptor
    rows: tuple       # [rows, cols]
    stats: tuple      # [2, rows]
    workspace: int    # bytes of the backward's workspace
    w_dtype: object
    keep: object      # the descriptor


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as [rows, cols] with contiguous columns (a view wherever the strides allow one)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


@_plan
def _norm_plan(rows, cols, x_dtype, z_dtype, w_dtype, index, eps, x_stride, res_stride, dy_stride=0,
               dz_stride=0) -> _NormPlan:
    if not 1 <= cols <= _lib.NORM_MAX_COLS:
        raise ValueError(f"the last axis must be 1 to {_lib.NORM_MAX_COLS} wide, got {cols}")
    d = _lib.NormDesc(rows, cols, _DTYPES[x_dtype], _DTYPES[z_dtype], _DTYPES[w_dtype], index, eps, x_stride,
                      res_stride, dy_stride, dz_stride)
    nbytes = ctypes.c_size_t(0)
    _lib.check(_lib.load().plstm_layer_norm_backward_workspace_size(_byref(d), _byref(nbytes)))
    return _NormPlan(_byref(d), (rows, cols), (2, rows), nbytes.value, w_dtype, d)


def _norm_inputs(x, residual, weight, bias, eps):
    """Checks the arguments; x and residual as rows, contiguous weights, and their plan."""
    if x.dim() == 0:
        raise ValueError("x must have at least one axis")
    cols, dev, dtype = x.shape[-1], x.device, x.dtype
    w_dtype = None
    if weight is not None:
        w_dtype = weight.dtype
        weight = _check_weight(weight, "weight", dev, dtype, cols)
    if bias is not None:
        if w_dtype is not None and bias.dtype is not w_dtype:
            raise ValueError("weight and bias must have one dtype")
        w_dtype = bias.dtype
        bias = _check_weight(bias, "bias", dev, dtype, cols)
    x2 = _rows(x) if cols else x.reshape(0, 0)
    r2 = None if residual is None else _rows(residual)
    plan = _norm_plan(x2.shape[0], cols, dtype, dtype if r2 is None else r2.dtype, w_dtype or dtype, dev.index, eps,
                      x2.stride(0), 0 if r2 is None else r2.stride(0))
    return x2, r2, weight, bias, plan


def _check_weight(w: torch.Tensor, name: str, dev: torch.device, dtype: torch.dtype, cols: int) -> torch.Tensor:
    if w.dim() != 1 or w.shape[0] != cols or w.device != dev:
        raise ValueError(f"{name} must be [{cols}] on {dev}, got {tuple(w.shape)} on {w.device}")
    if w.dtype is not dtype and w.dtype is not _F32:
        raise ValueError(f"{name} must be {dtype} or float32, got {w.dtype}")
    return w.contiguous()


def _shape(x, plan) -> tuple:
    """x's shape (as a tuple: torch.empty takes 1 us more for a torch.Size)."""
    return plan.rows if x.dim() == 2 else tuple(x.shape)


def _norm_forward(x, residual, weight, bias, plan, drop, keep, shape):
    """x, residual [rows, cols] -> (y, z or None, stats or None), y and z of the given shape."""
    dev = x.device
    y = _empty(shape, dtype=x.dtype, device=dev)
    z = None if residual is None else _empty(shape, dtype=residual.dtype, device=dev)
    stats = _empty(plan.stats, dtype=_F32, device=dev) if keep else None
    rc = _lib.load().plstm_layer_norm_forward(
        plan.desc, None if drop is None else _byref(drop), x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(bias),
        _ptr(z), y.data_ptr(), _ptr(stats), _stream(dev.index))
    if rc:
        _lib.check(rc)
    return y, z, stats


def _norm_backward(v, weight, stats, dy, dz, eps, drop, x_dtype, w_dtype, need):
    """Gradients of (x, residual, weight, bias) as `need` asks; drop is None for the plain norm."""
    dev = v.device
    shape = v.shape
    rows, cols = shape
    plan = _norm_plan(rows, cols, x_dtype, v.dtype, w_dtype, dev.index, eps, v.stride(0), 0, dy.stride(0),
                      0 if dz is None else dz.stride(0))
    dx = _empty(shape, dtype=x_dtype, device=dev) if need[0] else None
    dres = _empty(shape, dtype=v.dtype, device=dev) if need[1] else None
    dw = _empty(cols, dtype=w_dtype, device=dev) if need[2] else None
    db = _empty(cols, dtype=w_dtype, device=dev) if need[3] else None
    ws = _empty(plan.workspace + 16, dtype=torch.uint8, device=dev) if need[2] or need[3] else None
    rc = _lib.load().plstm_layer_norm_backward(
        plan.desc, None if drop is None else _byref(drop), drop is not None, dy.data_ptr(), _ptr(dz), v.data_ptr(),
        _ptr(weight), stats.data_ptr(), _ptr(dx), _ptr(dres), _ptr(dw), _ptr(db), _ptr(ws), plan.workspace,
        _stream(dev.index))
    if rc:
        _lib.check(rc)
    return dx, dres, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, how):
        plan, eps = how
        rows = _rows(x)
        # Not a view of rows: autograd refuses in-place operations on a view that a function returns.
        y, _, stats = _norm_forward(rows, None, weight, bias, plan, None, True, _shape(x, plan))
        ctx.save_for_backward(rows, weight, stats)
        ctx.args = (eps, plan.w_dtype)
        return y

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        eps, w_dtype = ctx.args
        need = ctx.needs_input_grad
        dx, _, dw, db = _norm_backward(x, weight, stats, _rows(dy), None, eps, None, x.dtype, w_dtype,
                                       (need[0], False, need[1], need[2]))
        return dx if dx is None or dy.dim() == 2 else dx.view(dy.shape), dw, db, None


class _DropoutAddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, how):
        plan, drop, seed, eps = how
        y, z, stats = _norm_forward(_rows(x), _rows(residual), weight, bias, plan, drop, True,
                                    _shape(x, plan))
        ctx.save_for_backward(z, weight, stats, seed)
        ctx.args = (drop, eps, x.dtype, plan.w_dtype)
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    @_first_order
    def backward(ctx, dy, dz):
        z, weight, stats, seed = ctx.saved_tensors
        drop, eps, x_dtype, w_dtype = ctx.args
        if dy is None and dz is None:
            return (None,) * 5
        shape = z.shape
        z = _rows(z)
        dy = torch.zeros((1, z.shape[1]), dtype=x_dtype, device=z.device).expand(z.shape) if dy is None else _rows(dy)
        dx, dres, dw, db = _norm_backward(z, weight, stats, dy, None if dz is None else _rows(dz), eps,
                                          _saved_drop(drop, seed), x_dtype, w_dtype, ctx.needs_input_grad)
        if len(shape) != 2:
            dx = None if dx is None else dx.view(shape)
            dres = None if dres is None else dres.view(shape)
        return dx, dres, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis, in x's type.

    weight and bias: x's type or f32.  Statistics, and the sums behind the weights' gradients,
    are f32.  Differentiable in x, weight and bias.
    """
    _refuse_transforms(x, weight, bias)
    x = _cuda_float(x, "x")
    rows, _, weight, bias, plan = _norm_inputs(x, None, weight, bias, eps)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, (plan, eps))
    return _norm_forward(rows, None, weight, bias, plan, None, False, _shape(x, plan))[0]


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                           bias: Optional[torch.Tensor] = None, p: float = 0.0,
                           seed: Union[int, torch.Tensor] = 0, offset: int = 0, *,
                           eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """The residual step in one pass: z = residual + dropout(x), y = layer_norm(z) -> (y, z).

    z is dropout(x, p, seed, offset, residual=residual) bit for bit, and y the norm of that stored
    z: with a residual of x's type, and rows that start on 16 bytes or are no multiple of eight
    wide, layer_norm(z, weight, bias, eps) bit for bit; else its sums may run in another order.
    The residual stream may be f32 under a 16-bit x; z has its type, y has x's.
    Differentiable in x, residual, weight and bias.
    """
    _refuse_transforms(x, residual, weight, bias)
    x = _cuda_float(x, "x")
    residual = _cuda_float(residual, "residual")
    _check_residual(residual, x)
    x2, r2, weight, bias, plan = _norm_inputs(x, residual, weight, bias, eps)
    drop = _drop_desc(p, seed, offset, x.device)
    if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad or
                                    (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _DropoutAddLayerNorm.apply(x, residual, weight, bias,
                                          (plan, drop, seed if isinstance(seed, torch.Tensor) else None, eps))
    return _norm_forward(x2, r2, weight, bias, plan, drop, False, _shape(x, plan))[:2]
