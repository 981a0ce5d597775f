"""ctypes binding of ``libcc1d_b200.so`` (the C ABI in ``include/causal_conv1d_b200.h``).

Every call launches on the current PyTorch stream of the tensors' device, under a device
guard, and returns without synchronising.  There is no CPU fallback: if the library is
missing or a tensor is not on a CUDA device, the call raises.
"""

from __future__ import annotations

import ctypes
import os
import struct
import threading

import torch

LIB_NAME = "libcc1d_b200.so"
LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), LIB_NAME)

_DTYPES = {
    torch.float32: 0,
    torch.float16: 1,
    torch.bfloat16: 2,
    torch.int32: 3,
    torch.int64: 4,
}

c_i32, c_i64, c_void_p = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


class CTensor(ctypes.Structure):
    _fields_ = [("data", c_void_p), ("dtype", c_i32), ("reserved", c_i32), ("stride", c_i64 * 3)]


class FwdParams(ctypes.Structure):
    _fields_ = [
        ("batch", c_i64), ("dim", c_i64), ("seqlen", c_i64), ("width", c_i64),
        ("x", CTensor), ("weight", CTensor), ("bias", CTensor), ("seq_idx", CTensor),
        ("initial_states", CTensor), ("final_states", CTensor), ("out", CTensor),
        ("silu", c_i32), ("reserved", c_i32),
    ]


class BwdParams(ctypes.Structure):
    _fields_ = [
        ("batch", c_i64), ("dim", c_i64), ("seqlen", c_i64), ("width", c_i64),
        ("x", CTensor), ("weight", CTensor), ("bias", CTensor), ("seq_idx", CTensor),
        ("initial_states", CTensor), ("dout", CTensor), ("dfinal_states", CTensor),
        ("dx", CTensor), ("dinitial_states", CTensor),
        ("dweight", c_void_p), ("dbias", c_void_p), ("workspace", c_void_p),
        ("workspace_bytes", c_i64), ("silu", c_i32), ("reserved", c_i32),
    ]


class UpdateParams(ctypes.Structure):
    _fields_ = [
        ("batch", c_i64), ("dim", c_i64), ("seqlen", c_i64), ("width", c_i64),
        ("state_batch", c_i64), ("state_len", c_i64),
        ("x", CTensor), ("conv_state", CTensor), ("weight", CTensor), ("bias", CTensor),
        ("cache_seqlens", CTensor), ("conv_state_indices", CTensor), ("out", CTensor),
        ("silu", c_i32), ("reserved", c_i32),
    ]


class VarlenParams(ctypes.Structure):
    _fields_ = [
        ("batch", c_i64), ("dim", c_i64), ("state_len", c_i64), ("total_tokens", c_i64),
        ("x", CTensor), ("cu_seqlens", CTensor), ("states", CTensor),
    ]


class FwdVarlenStatesParams(ctypes.Structure):
    _fields_ = [
        ("fwd", FwdParams), ("nseq", c_i64), ("state_len", c_i64),
        ("cu_seqlens", CTensor), ("states", CTensor),
    ]


# Bytes of the library's static backward scratch array (CC1D_STATIC_SCRATCH_BYTES).
STATIC_SCRATCH_BYTES = 32 * 1024 * 1024

# symbol -> (restype, argtypes); the same list is checked by the CPU test suite
SIGNATURES = {
    "cc1d_fwd_launch": (c_i32, [ctypes.POINTER(FwdParams), c_void_p]),
    "cc1d_bwd_workspace_bytes": (c_i64, [ctypes.POINTER(BwdParams)]),
    "cc1d_bwd_launch": (c_i32, [ctypes.POINTER(BwdParams), c_void_p]),
    "cc1d_bwd_launch_static": (c_i32, [ctypes.POINTER(BwdParams), c_void_p]),
    "cc1d_update_launch": (c_i32, [ctypes.POINTER(UpdateParams), c_void_p]),
    "cc1d_varlen_states_launch": (c_i32, [ctypes.POINTER(VarlenParams), c_void_p]),
    "cc1d_fwd_varlen_states_launch": (c_i32, [ctypes.POINTER(FwdVarlenStatesParams), c_void_p]),
    # the params of these are packed as flat 64-bit words (_words)
    "cc1d_recurrence_fwd_launch": (c_i32, [c_void_p, c_void_p]),
    "cc1d_recurrence_bwd_workspace_bytes": (c_i64, [c_void_p]),
    "cc1d_recurrence_bwd_launch": (c_i32, [c_void_p, c_void_p]),
    "cc1d_recurrence_update_launch": (c_i32, [c_void_p, c_void_p]),
    "cc1d_add_norm_fwd_launch": (c_i32, [c_void_p, c_void_p]),
    "cc1d_add_norm_bwd_workspace_bytes": (c_i64, [c_void_p]),
    "cc1d_add_norm_bwd_launch": (c_i32, [c_void_p, c_void_p]),
    "cc1d_last_error": (ctypes.c_char_p, []),
    "cc1d_status_string": (ctypes.c_char_p, [c_i32]),
    "cc1d_abi_version": (c_i32, []),
    "cc1d_launch_count": (c_i64, []),
}

_ERRORS = {1: ValueError, 2: TypeError, 3: NotImplementedError, 4: RuntimeError}

_lib = None
_lock = threading.Lock()


def load_library(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load (once) and return the C-ABI library; raise ImportError if it is absent."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(path):
                raise ImportError(
                    f"{path} is missing: build it with `python cute-causal-conv1d_b200/cc1d_build.py` "
                    "(nvcc, sm_100a). causal_conv1d has no CPU fallback."
                )
            lib = ctypes.CDLL(path)
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            _lib = lib
    return _lib


def _ct(t: torch.Tensor | None) -> CTensor:
    if t is None:
        return CTensor()
    try:
        code = _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}") from None
    s = list(t.stride()) + [0] * (3 - t.dim())
    return CTensor(t.data_ptr(), code, 0, (c_i64 * 3)(*s[:3]))


def _check(status: int) -> None:
    if status != 0:
        msg = load_library().cc1d_last_error().decode()
        raise _ERRORS.get(status, RuntimeError)(msg or f"causal_conv1d error {status}")


def _expect(name: str, t: torch.Tensor | None, shape: tuple) -> None:
    """Reject a tensor whose shape is not the one the kernels will index.  The C ABI
    receives pointers and strides only, so a tensor that is too small would otherwise be
    read or written out of bounds."""
    if t is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _expect_dims(name: str, t: torch.Tensor, ndim: int) -> None:
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got shape {tuple(t.shape)}")


def _conv_shapes(x, weight, bias, seq_idx, initial_states):
    """(batch, dim, seqlen, width) of a conv call after checking its input shapes."""
    _expect_dims("x", x, 3)
    _expect_dims("weight", weight, 2)
    B, D, L = x.shape
    W = weight.shape[1]
    _expect("weight", weight, (D, W))
    _expect("bias", bias, (D,))
    _expect("seq_idx", seq_idx, (B, L))
    _expect("initial_states", initial_states, (B, D, W - 1))
    return B, D, L, W


def _device_of(*tensors: torch.Tensor | None) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("causal_conv1d needs CUDA tensors (there is no CPU implementation)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"all tensors must be on one device ({dev} vs {t.device})")
    return dev


class _Guard:
    """Make ``device`` current for the launch (cheap when it already is)."""

    __slots__ = ("dev", "prev")

    def __init__(self, dev: torch.device):
        self.dev = dev.index if dev.index is not None else torch.cuda.current_device()
        self.prev = None

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.dev:
            self.prev = cur
            torch.cuda.set_device(self.dev)
        return torch.cuda.current_stream(self.dev).cuda_stream

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)
        return False


def fwd(x, weight, bias, seq_idx, initial_states, final_states, out, silu: bool) -> None:
    B, D, L, W = _conv_shapes(x, weight, bias, seq_idx, initial_states)
    _expect("final_states", final_states, (B, D, W - 1))
    _expect("out", out, (B, D, L))
    lib = load_library()
    dev = _device_of(x, weight, bias, seq_idx, initial_states, final_states, out)
    p = FwdParams(
        x.shape[0], x.shape[1], x.shape[2], weight.shape[1],
        _ct(x), _ct(weight), _ct(bias), _ct(seq_idx), _ct(initial_states),
        _ct(final_states), _ct(out), int(bool(silu)), 0,
    )
    with _Guard(dev) as stream:
        _check(lib.cc1d_fwd_launch(ctypes.byref(p), stream))


def _bwd_params(x, weight, bias, dout, seq_idx, initial_states, dfinal_states, dx, dinitial_states,
                dweight_f32, dbias_f32, silu: bool):
    B, D, L, W = _conv_shapes(x, weight, bias, seq_idx, initial_states)
    for name, t in (("dout", dout), ("dx", dx)):
        _expect(name, t, (B, D, L))
    for name, t in (("dfinal_states", dfinal_states), ("dinitial_states", dinitial_states)):
        _expect(name, t, (B, D, W - 1))
    _expect("dweight", dweight_f32, (D, W))
    _expect("dbias", dbias_f32, (D,))
    dev = _device_of(x, weight, bias, dout, seq_idx, initial_states, dfinal_states, dx,
                     dinitial_states, dweight_f32, dbias_f32)
    p = BwdParams(
        x.shape[0], x.shape[1], x.shape[2], weight.shape[1],
        _ct(x), _ct(weight), _ct(bias), _ct(seq_idx), _ct(initial_states), _ct(dout),
        _ct(dfinal_states), _ct(dx), _ct(dinitial_states),
        dweight_f32.data_ptr(), dbias_f32.data_ptr() if dbias_f32 is not None else None,
        None, 0, int(bool(silu)), 0,
    )
    return p, dev


def bwd_workspace_bytes(x, weight, bias, dout, seq_idx, initial_states, dfinal_states, dx,
                        dinitial_states, dweight_f32, dbias_f32, silu: bool) -> int:
    """Device scratch bytes ``bwd`` needs for these arguments (``cc1d_bwd_workspace_bytes``),
    so that a caller can allocate it once and pass it to every call."""
    p, _ = _bwd_params(x, weight, bias, dout, seq_idx, initial_states, dfinal_states, dx,
                       dinitial_states, dweight_f32, dbias_f32, silu)
    lib = load_library()
    need = lib.cc1d_bwd_workspace_bytes(ctypes.byref(p))
    if need < 0:
        _check(lib.cc1d_bwd_launch(ctypes.byref(p), None))  # raises with the message
    return int(need)


def bwd(x, weight, bias, dout, seq_idx, initial_states, dfinal_states, dx, dinitial_states,
        dweight_f32, dbias_f32, silu: bool, workspace: torch.Tensor | None = None) -> None:
    p, dev = _bwd_params(x, weight, bias, dout, seq_idx, initial_states, dfinal_states, dx,
                         dinitial_states, dweight_f32, dbias_f32, silu)
    lib = load_library()
    need = lib.cc1d_bwd_workspace_bytes(ctypes.byref(p))
    if need < 0:
        _check(lib.cc1d_bwd_launch(ctypes.byref(p), None))  # raises with the message
    if need > 0:
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        p.workspace = workspace.data_ptr()
        p.workspace_bytes = workspace.numel()
    with _Guard(dev) as stream:
        _check(lib.cc1d_bwd_launch(ctypes.byref(p), stream))


def update(x, conv_state, weight, bias, cache_seqlens, conv_state_indices, out, silu: bool) -> None:
    B, D, T, W = _conv_shapes(x, weight, bias, None, None)
    _expect_dims("conv_state", conv_state, 3)
    if conv_state.shape[1] != D:
        raise ValueError(f"conv_state must have dim {D} in its second dimension, got shape {tuple(conv_state.shape)}")
    _expect("cache_seqlens", cache_seqlens, (B,))
    _expect("conv_state_indices", conv_state_indices, (B,))
    _expect("out", out, (B, D, T))
    lib = load_library()
    dev = _device_of(x, conv_state, weight, bias, cache_seqlens, conv_state_indices, out)
    p = UpdateParams(
        x.shape[0], x.shape[1], x.shape[2], weight.shape[1], conv_state.shape[0], conv_state.shape[2],
        _ct(x), _ct(conv_state), _ct(weight), _ct(bias), _ct(cache_seqlens),
        _ct(conv_state_indices), _ct(out), int(bool(silu)), 0,
    )
    with _Guard(dev) as stream:
        _check(lib.cc1d_update_launch(ctypes.byref(p), stream))


def varlen_states(x, cu_seqlens, states) -> None:
    _expect_dims("x", x, 2)
    _expect_dims("cu_seqlens", cu_seqlens, 1)
    _expect_dims("states", states, 3)
    _expect("states", states, (cu_seqlens.shape[0] - 1, x.shape[1], states.shape[2]))
    lib = load_library()
    dev = _device_of(x, cu_seqlens, states)
    p = VarlenParams(states.shape[0], x.shape[1], states.shape[2], x.shape[0],
                     _ct(x), _ct(cu_seqlens), _ct(states))
    with _Guard(dev) as stream:
        _check(lib.cc1d_varlen_states_launch(ctypes.byref(p), stream))


def fwd_varlen_states(x, weight, bias, seq_idx, cu_seqlens, states, out, silu: bool) -> None:
    B, D, L, W = _conv_shapes(x, weight, bias, seq_idx, None)
    _expect("out", out, (B, D, L))
    _expect_dims("cu_seqlens", cu_seqlens, 1)
    _expect_dims("states", states, 3)
    _expect("states", states, (cu_seqlens.shape[0] - 1, D, states.shape[2]))
    lib = load_library()
    dev = _device_of(x, weight, bias, seq_idx, cu_seqlens, states, out)
    f = FwdParams(
        x.shape[0], x.shape[1], x.shape[2], weight.shape[1],
        _ct(x), _ct(weight), _ct(bias), _ct(seq_idx), _ct(None), _ct(None), _ct(out), int(bool(silu)), 0,
    )
    p = FwdVarlenStatesParams(f, states.shape[0], states.shape[2], _ct(cu_seqlens), _ct(states))
    with _Guard(dev) as stream:
        _check(lib.cc1d_fwd_varlen_states_launch(ctypes.byref(p), stream))


# ------------------------------------------------- recurrent-block operators
# Their params structs are made of 64-bit words only (a cc1d_tensor is five: data, dtype
# with the reserved half zero, three strides), so one struct.pack fills them, and the
# checks below are written for few Python operations: a decode step is short enough for the
# host's time per call to count.
RECURRENCE_CHUNK = 32  # CC1D_RECURRENCE_CHUNK
_NONE = (0, 0, 0, 0, 0)
_PAD = ((0, 0, 0), (0, 0), (0,), ())
_NO_GRADIENTS = _NONE * 6 + (0,)  # the recurrence's dout .. dinitial_states and dbias
RECURRENCE_PARAMS = struct.Struct("<78q")
RECURRENCE_UPDATE_PARAMS = struct.Struct("<39q")
ADD_NORM_PARAMS = struct.Struct("<55q2d")
_RECURRENCE_SCRATCH = struct.Struct("<2q")  # the last words: workspace, workspace_bytes
_ADD_NORM_SCRATCH = struct.Struct("<2q2d")  # ... and eps, dropout_p


def _words(t: torch.Tensor | None) -> tuple:
    if t is None:
        return _NONE
    s = t.stride()
    try:
        return (t.data_ptr(), _DTYPES[t.dtype], *s, *_PAD[len(s)])
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}") from None


def _check_all(tensors) -> int:
    """The device index of (name, tensor, shape) triples after checking the shapes (as
    ``_expect``) and that all are on one CUDA device.  The first must be there."""
    dev = tensors[0][1].get_device()
    same = dev >= 0
    for name, t, shape in tensors:
        if t is not None:
            if t.shape != shape:
                raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
            same = same and t.get_device() == dev
    if not same:
        _device_of(*(t for _, t, _ in tensors))  # raises with the reason
    return dev


class _DeviceStream:
    """The current stream's handle on device ``index``, which is current meanwhile."""

    __slots__ = ("index", "prev")

    def __init__(self, index: int):
        self.index = index

    def __enter__(self):
        self.prev = torch._C._cuda_getDevice()
        if self.prev != self.index:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.prev != self.index:
            torch.cuda.set_device(self.prev)
        return False


def _recurrence_states(batch, seq_idx, states) -> int:
    """Rows of the states: the batch's, or with packed sequences as many as the first of
    them has (0 if there are none)."""
    if seq_idx is None:
        return batch
    for t in states:
        if t is not None:
            return t.shape[0]
    return 0


def recurrence_fwd(x, gate, z, bias, seq_idx, initial_states, final_states, checkpoints, out) -> None:
    shape = x.shape
    if len(shape) != 3:
        _expect_dims("x", x, 3)
    B, D, L = shape
    dev = x.get_device()
    # absent tensors cost nothing here; `same` stays true while all are on x's device
    same = dev >= 0 and gate.get_device() == dev and out.get_device() == dev
    if gate.shape != shape or out.shape != shape:
        _expect("gate", gate, shape)
        _expect("out", out, shape)
    if z is not None:
        _expect("z", z, shape)
        same = same and z.get_device() == dev
    if bias is not None:
        _expect("gate_bias", bias, (D,))
        same = same and bias.get_device() == dev
    if seq_idx is not None:
        _expect("seq_idx", seq_idx, (B, L))
        same = same and seq_idx.get_device() == dev
    n = _recurrence_states(B, seq_idx, (initial_states, final_states))
    if initial_states is not None:
        _expect("initial_states", initial_states, (n, D))
        same = same and initial_states.get_device() == dev
    if final_states is not None:
        _expect("final_states", final_states, (n, D))
        same = same and final_states.get_device() == dev
    if checkpoints is not None:
        _expect("checkpoints", checkpoints, (B, -(-L // RECURRENCE_CHUNK), D))
        same = same and checkpoints.get_device() == dev
    if not same:
        _device_of(x, gate, z, bias, seq_idx, initial_states, final_states, checkpoints, out)
    p = RECURRENCE_PARAMS.pack(
        B, D, L, n, *_words(x), *_words(gate), *_words(z), *_words(bias), *_words(seq_idx), *_words(initial_states),
        *_words(final_states), *_words(out), *_NO_GRADIENTS, 0 if checkpoints is None else checkpoints.data_ptr(), 0, 0)
    lib = _lib or load_library()
    with _DeviceStream(dev) as stream:
        status = lib.cc1d_recurrence_fwd_launch(p, stream)
        if status:
            _check(status)


def recurrence_bwd(x, gate, z, bias, seq_idx, initial_states, checkpoints, dout, dfinal_states, dx, dgate, dz,
                   dinitial_states, dbias) -> None:
    _expect_dims("x", x, 3)
    shape = x.shape
    B, D, L = shape
    n = _recurrence_states(B, seq_idx, (initial_states, dfinal_states, dinitial_states))
    dev = _check_all((("x", x, shape), ("gate", gate, shape), ("z", z, shape), ("gate_bias", bias, (D,)),
                      ("seq_idx", seq_idx, (B, L)), ("initial_states", initial_states, (n, D)),
                      ("dout", dout, shape), ("dfinal_states", dfinal_states, (n, D)), ("dx", dx, shape),
                      ("dgate", dgate, shape), ("dz", dz, shape), ("dinitial_states", dinitial_states, (n, D)),
                      ("dbias", dbias, (D,)), ("checkpoints", checkpoints, (B, -(-L // RECURRENCE_CHUNK), D))))
    p = RECURRENCE_PARAMS.pack(
        B, D, L, n, *_words(x), *_words(gate), *_words(z), *_words(bias), *_words(seq_idx), *_words(initial_states),
        *_NONE * 2, *_words(dout), *_words(dfinal_states), *_words(dx), *_words(dgate), *_words(dz),
        *_words(dinitial_states), 0 if dbias is None else dbias.data_ptr(), checkpoints.data_ptr(), 0, 0)
    lib = _lib or load_library()
    with _DeviceStream(dev) as stream:
        need = lib.cc1d_recurrence_bwd_workspace_bytes(p)
        if need > 0:
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
            p = p[:-16] + _RECURRENCE_SCRATCH.pack(workspace.data_ptr(), need)
        status = lib.cc1d_recurrence_bwd_launch(p, stream)
        if status:
            _check(status)


def recurrence_update(x, gate, z, bias, state, state_indices, out) -> None:
    """x, gate, z, out: (batch, dim) or (batch, dim, tokens)."""
    shape = x.shape
    if len(shape) == 2:
        B, D = shape
        T = 1
    else:
        _expect_dims("x", x, 3)
        B, D, T = shape
    _expect_dims("state", state, 2)
    n = B if state_indices is None else state.shape[0]
    dev = _check_all((("x", x, shape), ("gate", gate, shape), ("z", z, shape), ("gate_bias", bias, (D,)),
                      ("state", state, (n, D)), ("state_indices", state_indices, (B,)), ("out", out, shape)))
    p = RECURRENCE_UPDATE_PARAMS.pack(
        B, D, T, n, *_words(x), *_words(gate), *_words(z), *_words(bias), *_words(state), *_words(state_indices),
        *_words(out))
    lib = _lib or load_library()
    with _DeviceStream(dev) as stream:
        status = lib.cc1d_recurrence_update_launch(p, stream)
        if status:
            _check(status)


def add_norm_fwd(x, residual, weight, rng_state, out, residual_out, eps: float, dropout_p: float) -> None:
    _expect_dims("x", x, 2)
    shape = x.shape
    dev = _check_all((("x", x, shape), ("residual", residual, shape), ("weight", weight, (shape[1],)),
                      ("rng_state", rng_state, (2,)), ("out", out, shape), ("residual_out", residual_out, shape)))
    p = ADD_NORM_PARAMS.pack(
        *shape, *_words(x), *_words(residual), *_words(weight), *_words(rng_state), *_words(out),
        *_words(residual_out), *_NONE * 4, 0, 0, 0, eps, dropout_p)
    lib = _lib or load_library()
    with _DeviceStream(dev) as stream:
        status = lib.cc1d_add_norm_fwd_launch(p, stream)
        if status:
            _check(status)


def add_norm_bwd(x_dtype, residual_out, weight, rng_state, dout, dresidual_out, dx, dresidual, dweight,
                 eps: float, dropout_p: float) -> None:
    _expect_dims("residual_out", residual_out, 2)
    shape = residual_out.shape
    dev = _check_all((("residual_out", residual_out, shape), ("weight", weight, (shape[1],)),
                      ("rng_state", rng_state, (2,)), ("dout", dout, shape), ("dresidual_out", dresidual_out, shape),
                      ("dx", dx, shape), ("dresidual", dresidual, shape), ("dweight", dweight, (shape[1],))))
    p = ADD_NORM_PARAMS.pack(
        *shape, 0, _DTYPES[x_dtype], 0, 0, 0, *_NONE, *_words(weight), *_words(rng_state), *_NONE,
        *_words(residual_out), *_words(dout), *_words(dresidual_out), *_words(dx), *_words(dresidual),
        0 if dweight is None else dweight.data_ptr(), 0, 0, eps, dropout_p)
    lib = _lib or load_library()
    with _DeviceStream(dev) as stream:
        need = lib.cc1d_add_norm_bwd_workspace_bytes(p)
        if need > 0:
            workspace = torch.empty(need, dtype=torch.uint8, device=weight.device)
            p = p[:-32] + _ADD_NORM_SCRATCH.pack(workspace.data_ptr(), need, eps, dropout_p)
        status = lib.cc1d_add_norm_bwd_launch(p, stream)
        if status:
            _check(status)


def launch_count() -> int:
    """Kernel launches made through the library by this process."""
    return int(load_library().cc1d_launch_count())
