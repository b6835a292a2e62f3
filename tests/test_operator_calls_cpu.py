"""What the Python calls of the training and streaming operators hand to the library and to
autograd, on the CPU: a stand-in takes the library's place and reads the pointers it is given."""
from __future__ import annotations

import ctypes
import types

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from persistent_lstm_hip_b200 import GatedScanRegressor, _lib, ops


class StandIn:
    """Calls of the C ABI that note what they were given.  Dropout writes its seed into every element."""

    def __init__(self):
        self.seeds, self.lengths = [], []

    def plstm_gated_scan_checkpoint_size(self, desc, nbytes):
        nbytes._obj.value = 4096
        return 0

    def plstm_gated_scan_forward(self, desc, gates, lengths, c0, h, c_n, checkpoints, stream):
        if lengths:
            self.lengths.append(list((ctypes.c_int32 * desc._obj.batch).from_address(lengths)))
        return 0

    def plstm_dropout(self, drop, n, x, x_dtype, residual, y, y_dtype, device, stream):
        self.seeds.append(self._seed(drop))
        (ctypes.c_float * n).from_address(y)[:] = [float(self.seeds[-1])] * n
        return 0

    def plstm_layer_norm_forward(self, desc, drop, *rest):
        self.seeds.append(None if drop is None else self._seed(drop))
        return 0

    def plstm_layer_norm_backward_workspace_size(self, desc, nbytes):
        nbytes._obj.value = 256
        return 0

    def plstm_layer_norm_backward(self, desc, drop, *rest):
        self.seeds.append(None if drop is None else self._seed(drop))
        return 0

    @staticmethod
    def _seed(drop):
        d = drop._obj
        return ctypes.c_uint64.from_address(d.seed_ptr).value if d.seed_ptr else d.seed


@pytest.fixture
def stand_in(monkeypatch):
    lib = StandIn()
    # A CPU tensor's device has no index.
    numbered = lambda kind: lambda *fields: kind(*(0 if f is None else f for f in fields))
    monkeypatch.setattr(ops, "_lib", types.SimpleNamespace(
        load=lambda: lib, check=_lib.check, DropoutDesc=_lib.DropoutDesc, NormDesc=numbered(_lib.NormDesc),
        ScanDesc=numbered(_lib.ScanDesc), NORM_MAX_COLS=_lib.NORM_MAX_COLS))
    monkeypatch.setattr(ops, "_stream", lambda index: 0)
    monkeypatch.setattr(ops, "_cuda_float", lambda t, name: t if t.stride(-1) == 1 else t.contiguous())
    monkeypatch.setattr(ops, "_require_cuda", lambda t, name, device, dtype=None: t.contiguous())
    return lib


# ---- a tensor seed under saved-tensor hooks ----------------------------------------------------------
def _copies():
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t)


def test_dropout_backward_reads_the_seed_that_autograd_kept(stand_in):
    """Hooks that pack a copy: autograd neither holds the caller's seed nor watches its version."""
    x, seed = torch.zeros(8, requires_grad=True), torch.tensor([42])
    with _copies():
        y = ops.dropout(x, 0.5, seed)
    seed.add_(1)
    (dx,) = torch.autograd.grad(y, x, torch.ones(8))
    assert stand_in.seeds == [42, 42] and (dx == 42).all()


def test_fused_backward_reads_the_seed_that_autograd_kept(stand_in):
    x, res, seed = torch.zeros(2, 8, requires_grad=True), torch.zeros(2, 8), torch.tensor([42])
    with _copies():
        y, z = ops.dropout_add_layer_norm(x, res, None, None, 0.5, seed)
    seed.add_(1)
    torch.autograd.grad(y, x, torch.ones(2, 8))
    assert stand_in.seeds == [42, 42]


def test_an_int_seed_is_the_backwards_too(stand_in):
    x = torch.zeros(8, requires_grad=True)
    with _copies():
        y = ops.dropout(x, 0.5, 7)
    torch.autograd.grad(y, x, torch.ones(8))
    assert stand_in.seeds == [7, 7]


# ---- lengths --------------------------------------------------------------------------------------
@pytest.mark.parametrize("seq_major", [False, True])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16,
                                   torch.uint32, torch.uint64])
def test_lengths_of_any_type_are_clamped_not_wrapped(stand_in, dtype, seq_major):
    B, T = 4, 300
    top = torch.iinfo(dtype).max
    values = [0, 7, top, min(top, 2 ** 32 + 5)]
    ops.gated_scan(torch.zeros((T, B, 8) if seq_major else (B, T, 8)), lengths=torch.tensor(values, dtype=dtype),
                   seq_major=seq_major)
    # The kernel's own clamp completes what fits into int32.
    assert [min(max(v, 0), T) for v in stand_in.lengths[0]] == [min(v, T) for v in values]


def test_negative_lengths_are_zero(stand_in):
    values = [-1, -(2 ** 31) - 7, torch.iinfo(torch.int64).min]
    ops.gated_scan(torch.zeros(3, 5, 8), lengths=torch.tensor(values))
    assert all(v <= 0 for v in stand_in.lengths[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.complex64])
def test_lengths_that_are_no_integers_are_refused(stand_in, dtype):
    with pytest.raises(ValueError, match="lengths"):
        ops.gated_scan(torch.zeros(2, 5, 8), lengths=torch.ones(2, dtype=dtype))


# ---- writes into the caller's state --------------------------------------------------------------------
def test_step_in_place_raises_the_states_version(stand_in):
    """A graph that saved a state must not differentiate with the step's values."""
    c = torch.zeros(2, 4, requires_grad=True)
    state = c + 1
    loss = (state ** 2).sum()
    with torch.no_grad():
        ops.gated_scan_step(torch.zeros(2, 16), state, out_c=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_step_in_place_takes_inference_tensors(stand_in):
    with torch.inference_mode():
        c = torch.zeros(2, 4)
        assert ops.gated_scan_step(torch.zeros(2, 16), c, out_c=c)[1] is c
    assert ops.gated_scan_step(torch.zeros(2, 16), c, out_c=c)[1] is c


@pytest.mark.parametrize("which", ["gates", "c", "out_c"])
def test_step_in_place_refuses_what_autograd_records(stand_in, which):
    """Also an out_c of its own that requires a gradient: its graph would belong to other values."""
    t = dict(gates=torch.zeros(2, 16), c=torch.zeros(2, 4), out_c=torch.zeros(2, 4))
    t[which].requires_grad_(True)
    with pytest.raises(ValueError, match="differentiable"):
        ops.gated_scan_step(t["gates"], t["c"], out_c=t["out_c"])
    with torch.no_grad():
        ops.gated_scan_step(t["gates"], t["c"], out_c=t["out_c"])


# ---- forward mode ---------------------------------------------------------------------------------------
def _one_argument_calls():
    """(the call as a function of one argument, that argument) for every argument that could carry a derivative."""
    g, x, c, w = torch.zeros(2, 5, 16), torch.zeros(4, 16), torch.zeros(2, 4), torch.zeros(16)
    return {
        "scan gates": (ops.gated_scan, g),
        "scan c0": (lambda v: ops.gated_scan(g, v), c),
        "step gates": (lambda v: ops.gated_scan_step(v, c), g[:, 0].clone()),
        "step c": (lambda v: ops.gated_scan_step(g[:, 0], v), c),
        "step out_c": (lambda v: ops.gated_scan_step(g[:, 0], c, out_c=v), c),
        "norm x": (ops.layer_norm, x),
        "norm weight": (lambda v: ops.layer_norm(x, v), w),
        "norm bias": (lambda v: ops.layer_norm(x, None, v), w),
        "dropout x": (lambda v: ops.dropout(v, 0.5, 1), x),
        "dropout residual": (lambda v: ops.dropout(x, 0.5, 1, residual=v), x),
        "fused x": (lambda v: ops.dropout_add_layer_norm(v, x), x),
        "fused residual": (lambda v: ops.dropout_add_layer_norm(x, v), x),
        "fused weight": (lambda v: ops.dropout_add_layer_norm(x, x, v), w),
        "fused bias": (lambda v: ops.dropout_add_layer_norm(x, x, None, v), w),
    }


@pytest.mark.parametrize("name", list(_one_argument_calls()))
def test_forward_mode_is_refused(stand_in, name):
    """Grad mode says nothing about tangents: no_grad keeps them."""
    call, v = _one_argument_calls()[name]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(v.clone(), torch.ones_like(v))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        call(v)  # a level without tangents takes the call


def test_tangents_of_a_gradient_are_refused(stand_in):
    x = torch.zeros(4, 16, requires_grad=True)
    y = ops.dropout(x, 0.5, 1)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(4, 16), torch.ones(4, 16))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, dual)


# ---- tracing --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", list(_one_argument_calls()))
def test_tracing_is_refused(stand_in, name):
    """What a tracer records of these calls is their allocations: replaying it gives uninitialised memory, and of a
    recorded call a plan for one shape."""
    call, v = _one_argument_calls()[name]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, (v,), check_trace=False)
    with torch.no_grad(), pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, (v,), check_trace=False)
    for pre_dispatch in (False, True):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(lambda a: call(a), pre_dispatch=pre_dispatch)(v)
    call(v)


def test_tracing_a_backward_is_refused(stand_in):
    x = torch.zeros(4, 16, requires_grad=True)
    y = ops.dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda dy: torch.autograd.grad(y, x, dy))(torch.ones(4, 16))


# ---- in-place operations on results -----------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(16,), (4, 16), (2, 3, 16), (2, 2, 3, 16)])
def test_results_take_in_place_operations(stand_in, shape):
    """relu_ on a result in training, whatever its axes: no result is a view made inside a function."""
    x, w = torch.zeros(shape, requires_grad=True), torch.ones(16, requires_grad=True)
    y = ops.layer_norm(x, w)
    assert y.shape == shape
    y.relu_()
    assert torch.autograd.grad(y.sum(), (x, w))[0].shape == shape
    y, z = ops.dropout_add_layer_norm(x, torch.zeros(shape), w)
    assert y.shape == z.shape == shape
    y.relu_()
    assert torch.autograd.grad(y.sum() + z.sum(), (x, w))[0].shape == shape
    y = ops.dropout(x, 0.5, 1)
    y.relu_()
    assert torch.autograd.grad(y.sum(), x)[0].shape == shape


def test_scan_results_take_in_place_operations(stand_in):
    gates = torch.zeros(2, 5, 16, requires_grad=True)
    ops.gated_scan(gates)[0].relu_()
    h, c = ops.gated_scan_step(gates[:, 0], torch.zeros(2, 4))
    h.relu_()
    c.mul_(2)


def test_changing_the_saved_residual_stream_is_noticed(stand_in):
    """The backward needs z as it was."""
    x = torch.zeros(2, 3, 16, requires_grad=True)
    y, z = ops.dropout_add_layer_norm(x, torch.zeros(2, 3, 16))
    z.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- no rows ------------------------------------------------------------------------------------------------
def test_fused_step_without_rows_may_have_no_residual_pointer():
    """An empty tensor's pointer is NULL, and the call still the fused one (returns before any CUDA call)."""
    lib, drop = _lib.load(), ctypes.byref(_lib.DropoutDesc(0.5, 1, 0, None))
    for z_dtype in (_lib.F16, _lib.F32):
        d = ctypes.byref(_lib.NormDesc(0, 8, _lib.F16, z_dtype, _lib.F32, 0, 1e-5, 8, 8, 8, 8))
        assert lib.plstm_layer_norm_forward(d, drop, None, None, None, None, None, None, None, None) == 0
    d = ctypes.byref(_lib.NormDesc(1, 8, _lib.F16, _lib.F16, _lib.F32, 0, 1e-5, 8, 8, 8, 8))
    assert lib.plstm_layer_norm_forward(d, drop, 16, None, None, None, None, 16, None, None) == _lib.EINVAL
    assert "residual" in _lib.last_error()


# ---- sizes ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seq_major", [False, True])
@pytest.mark.parametrize("shape", [(2 ** 32 + 1, 1, 8), (1, 2 ** 32 + 1, 8), (2 ** 31, 1, 8), (1, 1, 2 ** 34 + 4)])
def test_scan_refuses_axes_beyond_its_descriptor(stand_in, shape, seq_major):
    """They would wrap in its 32-bit fields: 2^32 + 1 rows to one row."""
    strides = (shape[1] * shape[2], shape[2], 1)
    with pytest.raises(ValueError, match="below 2.31"):
        ops._scan_plan(shape, strides, torch.bfloat16, None, seq_major)


# ---- tensors without memory of their own --------------------------------------------------------------------
class Wrapper(torch.Tensor):
    """As DTensor and others are built: operations reach the inner tensor, data_ptr() is 0."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        args = [a.inner if isinstance(a, Wrapper) else a for a in args]
        return Wrapper(func(*args, **(kwargs or {})))


# The rest (gates, x, out_c) may not be left out, and the library refuses a NULL there.
_OPTIONAL = ("scan c0", "step c", "norm weight", "norm bias", "dropout residual", "fused residual", "fused weight",
             "fused bias")
_WRAPPED_CALLS = {
    **{name: _one_argument_calls()[name] for name in _OPTIONAL},
    "scan lengths": (lambda v: ops.gated_scan(torch.zeros(2, 5, 16), lengths=v), torch.tensor([1, 2], dtype=torch.int32)),
    "dropout seed": (lambda v: ops.dropout(torch.zeros(8), 0.5, v), torch.tensor([5])),
    "fused seed": (lambda v: ops.dropout_add_layer_norm(torch.zeros(2, 8), torch.zeros(2, 8), p=0.5, seed=v),
                   torch.tensor([5])),
}


@pytest.mark.parametrize("name", list(_WRAPPED_CALLS))
def test_tensors_without_memory_are_refused(stand_in, name):
    """Their NULL would read as no weight, no state, no residual, no lengths or the seed 0."""
    call, v = _WRAPPED_CALLS[name]
    wrapped = Wrapper(v.clone())
    assert wrapped.data_ptr() == 0
    with pytest.raises(ValueError, match="memory of its own"):
        call(wrapped)


# ---- states of the regressor ---------------------------------------------------------------------------------
@pytest.mark.parametrize("default", [torch.float32, torch.float64, torch.bfloat16])
def test_states_are_f32_whatever_the_default_type(default):
    m, before = GatedScanRegressor(3, 8, 2, 2), torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        state = m.init_state(4)
    finally:
        torch.set_default_dtype(before)
    assert [(c.dtype, tuple(c.shape)) for c in state] == [(torch.float32, (4, 8))] * 2
