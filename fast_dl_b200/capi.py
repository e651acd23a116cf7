"""ctypes binding of libfdl_kernels.so -- the same C ABI a cgo/JNI/C++ caller would bind.

This module is harness plumbing for the Python tests and bench: it declares the
prototypes of include/fdl_kernels.h, loads the in-tree library, and offers thin helpers
that take torch CUDA tensors (used only as device-memory handles: `data_ptr()` and the
current stream).  There is no fallback: if the library is missing or a call fails, an
exception is raised.
"""
from __future__ import annotations

import ctypes as C
from pathlib import Path

from . import build as _build

ADD, SUB, MUL, DIV = 0, 1, 2, 3
RELU, LEAKY_RELU, GELU, SIGMOID, TANH = 0, 1, 2, 3, 4
REDUCE_SUM, REDUCE_MEAN, REDUCE_MAX = 0, 1, 2
TREE_INTERLEAVE, TREE_ADDRESS = 0, 1
F32, F16, BF16 = 0, 1, 2
NORM_NONE, NORM_RMS, NORM_LAYER = 0, 1, 2
GATE_PLAIN, GATE_SIGMOID, GATE_TANH = 0, 1, 2

_vp, _i64, _int, _f32, _f64, _sz = C.c_void_p, C.c_int64, C.c_int, C.c_float, C.c_double, C.c_size_t
_pi64 = C.POINTER(C.c_int64)

# name -> (restype, argtypes); must list every symbol include/fdl_kernels.h declares.
PROTOTYPES = {
    "fdl_version": (_int, []),
    "fdl_error_string": (C.c_char_p, [_int]),
    "fdl_device_count": (_int, []),
    "fdl_set_device": (_int, [_int]),
    "fdl_stream_synchronize": (_int, [_vp]),
    "fdl_take_device_error": (_int, []),
    "fdl_set_tuning": (_int, [C.c_char_p, _int]),
    "fdl_debug_sum_trace": (_int, [C.POINTER(C.c_uint64)]),
    "fdl_binary_f32": (_int, [_vp, _vp, _vp, _i64, _int, _vp]),
    "fdl_unary_f32": (_int, [_vp, _vp, _i64, _int, _f32, _vp]),
    "fdl_mul_add_relu_f32": (_int, [_vp, _vp, _vp, _vp, _i64, _vp]),
    "fdl_add_row_bias_f32": (_int, [_vp, _vp, _i64, _i64, _vp]),
    "fdl_add_row_bias_relu_f32": (_int, [_vp, _vp, _i64, _i64, _vp]),
    "fdl_broadcast_binary_f32": (_int, [_vp, _vp, _vp, _int, _pi64, _pi64, _pi64, _int, _vp]),
    "fdl_block_reduce_1024_f32": (_int, [_vp, _vp, _i64, _int, _vp]),
    "fdl_sum_scratch_bytes": (_sz, [_i64]),
    "fdl_reduce_cols_scratch_bytes": (_sz, [_i64, _i64, _i64]),
    "fdl_sum_f32": (_int, [_vp, _i64, _vp, _vp, _vp, _sz, _vp]),
    "fdl_sum_f32_static": (_int, [_vp, _i64, _vp, _vp, _vp]),
    "fdl_debug_split_ticket": (_int, [_i64, _i64, _i64, C.c_uint, C.POINTER(C.c_int64), C.POINTER(C.c_int),
                                      C.POINTER(C.c_int)]),
    "fdl_exchange_create": (_int, [_int, _int, C.POINTER(C.c_void_p)]),
    "fdl_exchange_local_handle": (_int, [_vp, C.c_char_p]),
    "fdl_exchange_connect": (_int, [_vp, C.c_char_p]),
    "fdl_exchange_buffer": (_int, [_vp, C.POINTER(C.c_void_p)]),
    "fdl_exchange_connect_pointers": (_int, [_vp, C.POINTER(C.c_void_p)]),
    "fdl_exchange_destroy": (_int, [_vp]),
    "fdl_sum_allreduce_f32": (_int, [_vp, _i64, _vp, _vp, _vp, _vp, _sz, _vp]),
    "fdl_sum_allreduce_start_f32": (_int, [_vp, _i64, _vp, _vp, _sz, _vp]),
    "fdl_sum_allreduce_finish_f32": (_int, [_vp, _vp, _vp, _vp]),
    "fdl_reduce_cols_allreduce_f32": (_int, [_vp, _i64, _i64, _vp, _int, _f64, _vp, _vp, _sz, _vp]),
    "fdl_reduce_rows_f32": (_int, [_vp, _i64, _i64, _vp, _int, _vp]),
    "fdl_argmax_rows_f32": (_int, [_vp, _i64, _i64, _vp, _vp]),
    "fdl_reduce_cols_f32": (_int, [_vp, _i64, _i64, _i64, _vp, _int, _f64, _vp, _sz, _vp]),
    "fdl_softmax_rows_f32": (_int, [_vp, _vp, _i64, _i64, _vp]),
    "fdl_layernorm_rows_f32": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _f32, _vp]),
    "fdl_cross_entropy_f32": (_int, [_vp, _vp, _vp, _i64, _i64, _vp]),
    "fdl_transpose_f32": (_int, [_vp, _vp, _i64, _vp]),
    "fdl_uniform_f32": (_int, [_vp, _i64, _f32, _f32, C.c_uint64, _vp]),
    "fdl_normal_f32": (_int, [_vp, _i64, _f32, _f32, C.c_uint64, _vp]),
    "fdl_distill_topk": (_int, [_vp, _i64, _int, _vp, _int, _vp, _vp, _vp, _i64, _i64, _i64, _f32, _f32, _vp, _vp, _vp,
                                _vp]),
    "fdl_distill_topk_backward": (_int, [_vp, _i64, _int, _vp, _int, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _f32,
                                         _f32, _vp, _i64, _vp]),
    "fdl_distill_topk_with_grad": (_int, [_vp, _i64, _int, _vp, _int, _vp, _vp, _vp, _i64, _i64, _i64, _f32, _f32, _vp,
                                          _vp, _vp, _vp, _i64, _vp]),
    "fdl_norm_residual": (_int, [_vp, _vp, _vp, _i64, _int, _int, _vp, _vp, _int, _vp, _vp, _vp, _vp, _vp, _i64, _i64,
                                 _f32, _f32, _f32, _int, _vp]),
    "fdl_norm_residual_backward_scratch_bytes": (_sz, [_i64, _i64, _i64]),
    "fdl_norm_residual_backward": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _int, _int, _vp, _vp, _int, _vp, _vp, _vp,
                                          _vp, _vp, _vp, _vp, _vp, _i64, _i64, _f32, _f32, _int, _vp, _sz, _vp]),
    "fdl_verify_draft": (_int, [_vp, _i64, _i64, _vp, _i64, _i64, _int, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _vp, _vp,
                                _vp]),
    "fdl_host_binary_f32": (_int, [_vp, _vp, _vp, _i64, _int]),
    "fdl_host_unary_f32": (_int, [_vp, _vp, _i64, _int, _f32]),
    "fdl_host_mul_add_relu_f32": (_int, [_vp, _vp, _vp, _vp, _i64]),
    "fdl_host_row_broadcast_f32": (_int, [_vp, _vp, _vp, _i64, _i64, _int]),
    "fdl_host_sum_f32": (_int, [_vp, _i64, C.POINTER(C.c_double)]),
    "fdl_host_sweep_f32": (_int, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, C.POINTER(C.c_double)]),
}


class FdlError(RuntimeError):
    def __init__(self, status: int, text: str, where: str):
        super().__init__(f"{where}: {text} (status {status})")
        self.status = status


_lib = None


def library_path() -> Path:
    return _build.kernels_lib_path()


def lib() -> C.CDLL:
    """The loaded library with prototypes attached.  Raises if it has not been built."""
    global _lib
    if _lib is None:
        path = library_path()
        if not path.exists():
            raise FileNotFoundError(
                f"{path} is missing: run `python -m fast_dl_b200.build` (there is no fallback path)")
        handle = C.CDLL(str(path))
        for name, (restype, argtypes) in PROTOTYPES.items():
            fn = getattr(handle, name)  # AttributeError if the symbol is not exported
            fn.restype = restype
            fn.argtypes = argtypes
        _lib = handle
    return _lib


def check(status: int, where: str) -> None:
    if status != 0:
        raise FdlError(status, lib().fdl_error_string(status).decode(), where)


# ---- torch-tensor conveniences -------------------------------------------------------------


def _stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _require(t, dtype=None):
    import torch
    if not t.is_cuda or not t.is_contiguous():
        raise ValueError("expected a contiguous CUDA tensor")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"expected dtype {dtype}, got {t.dtype}")
    return t


def set_tuning(key: str, value: int) -> None:
    check(lib().fdl_set_tuning(key.encode(), value), f"fdl_set_tuning({key})")


def use_device(index: int) -> None:
    check(lib().fdl_set_device(index), "fdl_set_device")


def binary(a, b, op, out=None):
    import torch
    _require(a, torch.float32), _require(b, torch.float32)
    if a.numel() != b.numel():
        raise ValueError("binary: operands differ in size")
    out = torch.empty_like(a) if out is None else out
    check(lib().fdl_binary_f32(_ptr(a), _ptr(b), _ptr(out), a.numel(), op, _stream()), "fdl_binary_f32")
    return out


def unary(x, op, alpha=0.01, out=None):
    import torch
    _require(x, torch.float32)
    out = torch.empty_like(x) if out is None else out
    check(lib().fdl_unary_f32(_ptr(x), _ptr(out), x.numel(), op, alpha, _stream()), "fdl_unary_f32")
    return out


def mul_add_relu(a, b, c, out=None):
    import torch
    for t in (a, b, c):
        _require(t, torch.float32)
    out = torch.empty_like(a) if out is None else out
    check(lib().fdl_mul_add_relu_f32(_ptr(a), _ptr(b), _ptr(c), _ptr(out), a.numel(), _stream()),
          "fdl_mul_add_relu_f32")
    return out


def add_row_bias_(out, bias, relu=False):
    rows, cols = out.shape
    fn = lib().fdl_add_row_bias_relu_f32 if relu else lib().fdl_add_row_bias_f32
    check(fn(_ptr(out), _ptr(bias), rows, cols, _stream()), "fdl_add_row_bias_f32")
    return out


def broadcast_strides(shape, out_shape):
    """Element strides of a contiguous tensor of `shape` viewed as `out_shape` (0 = broadcast)."""
    nd = len(out_shape)
    shape = (1,) * (nd - len(shape)) + tuple(shape)
    strides, acc = [0] * nd, 1
    for i in range(nd - 1, -1, -1):
        if shape[i] == 1 and out_shape[i] != 1:
            strides[i] = 0
        elif shape[i] == out_shape[i]:
            strides[i] = acc if shape[i] != 1 else 0
        else:
            raise ValueError(f"shape {shape} does not broadcast to {out_shape}")
        acc *= shape[i]
    return strides


def broadcast_shape(sa, sb):
    nd = max(len(sa), len(sb))
    sa = (1,) * (nd - len(sa)) + tuple(sa)
    sb = (1,) * (nd - len(sb)) + tuple(sb)
    out = []
    for x, y in zip(sa, sb):
        if x != y and x != 1 and y != 1:
            raise ValueError(f"shapes {sa} and {sb} do not broadcast")
        out.append(max(x, y))
    return tuple(out)


def broadcast_binary(a, b, op, out=None):
    import torch
    _require(a, torch.float32), _require(b, torch.float32)
    oshape = broadcast_shape(tuple(a.shape), tuple(b.shape))
    out = torch.empty(oshape, dtype=torch.float32, device=a.device) if out is None else out
    nd = len(oshape)
    arr = C.c_int64 * nd
    check(lib().fdl_broadcast_binary_f32(
        _ptr(a), _ptr(b), _ptr(out), nd, arr(*oshape), arr(*broadcast_strides(a.shape, oshape)),
        arr(*broadcast_strides(b.shape, oshape)), op, _stream()), "fdl_broadcast_binary_f32")
    return out


def block_reduce_1024(x, tree=TREE_ADDRESS):
    import torch
    _require(x, torch.float32)
    out = torch.empty(x.numel() // 1024, dtype=torch.float32, device=x.device)
    check(lib().fdl_block_reduce_1024_f32(_ptr(x), _ptr(out), x.numel(), tree, _stream()),
          "fdl_block_reduce_1024_f32")
    return out


def full_sum(x, want_f64=False, scratch=None):
    import torch
    _require(x, torch.float32)
    out = torch.empty(1, dtype=torch.float32, device=x.device)
    out64 = torch.empty(1, dtype=torch.float64, device=x.device) if want_f64 else None
    check(lib().fdl_sum_f32(_ptr(x), x.numel(), _ptr(out), _ptr(out64), _ptr(scratch),
                            0 if scratch is None else scratch.numel() * scratch.element_size(),
                            _stream()), "fdl_sum_f32")
    return (out, out64) if want_f64 else out


def full_sum_static(x, want_f64=False):
    """fdl_sum_f32_static: the full sum with its scratch in the library's fixed device array."""
    import torch
    _require(x, torch.float32)
    out = torch.empty(1, dtype=torch.float32, device=x.device)
    out64 = torch.empty(1, dtype=torch.float64, device=x.device) if want_f64 else None
    check(lib().fdl_sum_f32_static(_ptr(x), x.numel(), _ptr(out), _ptr(out64), _stream()),
          "fdl_sum_f32_static")
    return (out, out64) if want_f64 else out


def reduce_rows(x, op):
    import torch
    _require(x, torch.float32)
    rows, cols = x.shape
    out = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(lib().fdl_reduce_rows_f32(_ptr(x), rows, cols, _ptr(out), op, _stream()), "fdl_reduce_rows_f32")
    return out


def argmax_rows(x):
    import torch
    _require(x, torch.float32)
    rows, cols = x.shape
    out = torch.empty(rows, dtype=torch.int64, device=x.device)
    check(lib().fdl_argmax_rows_f32(_ptr(x), rows, cols, _ptr(out), _stream()), "fdl_argmax_rows_f32")
    return out


def reduce_cols(x, op, mean_divisor=None, scratch=None):
    """x: [rows, cols] or [batch, rows, cols]; reduces over rows."""
    import torch
    _require(x, torch.float32)
    if x.dim() == 2:
        batch, (rows, cols) = 1, x.shape
        oshape = (cols,)
    else:
        batch, rows, cols = x.shape
        oshape = (batch, cols)
    out = torch.empty(oshape, dtype=torch.float32, device=x.device)
    div = float(rows if mean_divisor is None else mean_divisor)
    check(lib().fdl_reduce_cols_f32(_ptr(x), batch, rows, cols, _ptr(out), op, div, _ptr(scratch),
                                    0 if scratch is None else scratch.numel() * scratch.element_size(),
                                    _stream()), "fdl_reduce_cols_f32")
    return out


def softmax_rows(x, out=None):
    import torch
    _require(x, torch.float32)
    rows, cols = x.shape
    out = torch.empty_like(x) if out is None else out
    check(lib().fdl_softmax_rows_f32(_ptr(x), _ptr(out), rows, cols, _stream()), "fdl_softmax_rows_f32")
    return out


def layernorm_rows(x, gamma=None, beta=None, eps=1e-5, out=None, want_stats=False):
    import torch
    _require(x, torch.float32)
    rows, cols = x.shape
    out = torch.empty_like(x) if out is None else out
    mean = torch.empty(rows, dtype=torch.float32, device=x.device) if want_stats else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if want_stats else None
    check(lib().fdl_layernorm_rows_f32(_ptr(x), _ptr(gamma), _ptr(beta), _ptr(out), _ptr(mean), _ptr(rstd),
                                       rows, cols, eps, _stream()), "fdl_layernorm_rows_f32")
    return (out, mean, rstd) if want_stats else out


def cross_entropy(logits, labels):
    import torch
    _require(logits, torch.float32), _require(labels, torch.int64)
    batch, classes = logits.shape
    loss = torch.empty(1, dtype=torch.float32, device=logits.device)
    check(lib().fdl_cross_entropy_f32(_ptr(logits), _ptr(labels), _ptr(loss), batch, classes, _stream()),
          "fdl_cross_entropy_f32")
    return loss


def transpose(x):
    import torch
    _require(x, torch.float32)
    out = torch.empty_like(x)
    check(lib().fdl_transpose_f32(_ptr(x), _ptr(out), x.shape[0], _stream()), "fdl_transpose_f32")
    return out


def random_fill(n, normal, p0, p1, seed, device="cuda"):
    import torch
    out = torch.empty(n, dtype=torch.float32, device=device)
    fn = lib().fdl_normal_f32 if normal else lib().fdl_uniform_f32
    check(fn(_ptr(out), n, p0, p1, seed, _stream()), "fdl_random_fill")
    return out


def sum_trace() -> list:
    """The eight words left by the most recent full sum launched with the tuning key sum_trace set."""
    words = (C.c_uint64 * 8)()
    check(lib().fdl_debug_sum_trace(words), "fdl_debug_sum_trace")
    return list(words)


def take_device_error() -> None:
    check(lib().fdl_take_device_error(), "device-side wait")


# ---- training a model from a teacher, serving with a draft model ---------------------------------------
#
# 32-bit, 16-bit float and bfloat16 tensors on the current device; results go to new tensors (scratch
# too, so that a captured call replays on memory of its own).


# A call for one token or one sequence takes the GPU a few microseconds, so the checks are written to take few:
# one combined test a tensor, its parts told apart only when it fails.

_torch = None
_dtype_codes = {}
_raw_stream = None


def _load_torch():
    global _torch, _raw_stream
    import torch
    _dtype_codes.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    # the current stream's handle without a Stream object around it, where this torch has that
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda device: torch.cuda.current_stream(device).cuda_stream)
    _torch = torch
    return torch


def _device_of(where, t):
    """The current CUDA device, if `t` is on it."""
    torch = _torch or _load_torch()
    if t.is_cuda:
        device = torch.cuda.current_device()
        if t.get_device() == device:
            return device
    raise ValueError(f"{where}: expected tensors on the current CUDA device, got {t.device}")


def _dtype_code(where, t):
    code = _dtype_codes.get(t.dtype)
    if code is None:
        raise ValueError(f"{where}: expected float32, float16 or bfloat16, got {t.dtype}")
    return code


def _given(where, name, t, device, dtype, shape, contiguous=True):
    """The address of `t` (None for None), which has to be on `device`, of this type and shape."""
    if t is None:
        return None
    if t.get_device() == device and t.dtype is dtype and t.shape == shape and (not contiguous or t.is_contiguous()):
        return t.data_ptr()
    if t.get_device() != device:
        raise ValueError(f"{where}: {name}: expected a tensor on the current CUDA device, got {t.device}")
    if t.dtype is not dtype:
        raise ValueError(f"{where}: {name}: expected dtype {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{where}: {name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{where}: {name}: expected a contiguous tensor")


def _row_stride(where, name, t, rows, cols):
    """Row stride of a matrix whose rows are contiguous and do not overlap."""
    if t.is_contiguous():
        return cols
    between, within = t.stride()
    if (cols > 1 and within != 1) or (rows > 1 and between < cols):
        raise ValueError(f"{where}: {name}: expected contiguous rows that do not overlap, got strides {t.stride()}")
    return between if rows > 1 else cols


def _distill_args(where, logits, teacher, index, teacher_lse, row_weight, temperature, scale):
    device = _device_of(where, logits)
    torch = _torch
    if logits.dim() != 2 or index.dim() != 2:
        raise ValueError(f"{where}: expected logits [rows, vocab] and index [rows, k]")
    rows, vocab = logits.shape
    k = index.shape[1]
    row = (rows,)
    head = (logits.data_ptr(), _row_stride(where, "logits", logits, rows, vocab), _dtype_code(where, logits),
            _given(where, "teacher", teacher, device, teacher.dtype, (rows, k)), _dtype_code(where, teacher),
            _given(where, "index", index, device, torch.int64, (rows, k)),
            _given(where, "teacher_lse", teacher_lse, device, torch.float32, row),
            _given(where, "row_weight", row_weight, device, torch.float32, row))
    return device, head, (rows, vocab, k, temperature, 1.0 / max(rows, 1) if scale is None else scale)


def _grad_for(where, logits, out, device):
    rows, vocab = logits.shape
    if out is None:
        return _torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device), vocab
    _given(where, "out", out, device, logits.dtype, logits.shape, contiguous=False)
    return out, _row_stride(where, "out", out, rows, vocab)


def distill_topk(logits, teacher, index, teacher_lse=None, row_weight=None, temperature=1.0, scale=None):
    """Distillation loss on the teacher's k highest logits: (loss [1], row_loss [rows], row_stats [rows, 2]).

    logits [rows, vocab] (rows may be padded), teacher and index (int64) [rows, k]; an index outside
    [0, vocab) is padding.  scale: default 1 / rows (the mean).  row_stats goes to distill_topk_backward."""
    device, head, sizes = _distill_args("distill_topk", logits, teacher, index, teacher_lse, row_weight, temperature, scale)
    rows, f32 = sizes[0], _torch.float32
    loss = _torch.empty((1,), dtype=f32, device=logits.device)
    row_loss = _torch.empty((rows,), dtype=f32, device=logits.device)
    stats = _torch.empty((rows, 2), dtype=f32, device=logits.device)
    check(lib().fdl_distill_topk(*head, *sizes, loss.data_ptr(), row_loss.data_ptr(), stats.data_ptr(),
                                 _raw_stream(device)), "fdl_distill_topk")
    return loss, row_loss, stats


def distill_topk_backward(logits, teacher, index, row_stats, teacher_lse=None, row_weight=None, temperature=1.0,
                          scale=None, grad_loss=None, out=None):
    """Gradient of grad_loss * loss in the logits' type; out may be `logits` itself."""
    where = "distill_topk_backward"
    device, head, sizes = _distill_args(where, logits, teacher, index, teacher_lse, row_weight, temperature, scale)
    f32 = _torch.float32
    stats = _given(where, "row_stats", row_stats, device, f32, (sizes[0], 2))
    up = None if grad_loss is None else _given(where, "grad_loss", grad_loss.reshape(-1), device, f32, (1,))
    grad, stride = _grad_for(where, logits, out, device)
    check(lib().fdl_distill_topk_backward(*head, stats, up, *sizes, grad.data_ptr(), stride, _raw_stream(device)),
          "fdl_distill_topk_backward")
    return grad


def distill_topk_with_grad(logits, teacher, index, teacher_lse=None, row_weight=None, temperature=1.0, scale=None,
                           out=None):
    """(loss [1], row_loss [rows], gradient of the loss); out may be `logits` itself."""
    where = "distill_topk_with_grad"
    device, head, sizes = _distill_args(where, logits, teacher, index, teacher_lse, row_weight, temperature, scale)
    rows, f32 = sizes[0], _torch.float32
    loss = _torch.empty((1,), dtype=f32, device=logits.device)
    row_loss = _torch.empty((rows,), dtype=f32, device=logits.device)
    stats = _torch.empty((rows, 2), dtype=f32, device=logits.device)
    grad, stride = _grad_for(where, logits, out, device)
    check(lib().fdl_distill_topk_with_grad(*head, *sizes, loss.data_ptr(), row_loss.data_ptr(), stats.data_ptr(),
                                           grad.data_ptr(), stride, _raw_stream(device)), "fdl_distill_topk_with_grad")
    return loss, row_loss, grad


def norm_residual(x, h, post=NORM_RMS, pre=NORM_RMS, gate=None, gate_act=GATE_PLAIN, post_gamma=None, post_beta=None,
                  pre_gamma=None, pre_beta=None, residual_scale=1.0, block_scale=1.0, eps=1e-5, out=None, out_n=None):
    """y = residual_scale * x + block_scale * act(gate) * norm_post(h) and n = norm_pre(y): (y, n, stats [rows, 4]).

    gate: [gate_rows, cols], gate_rows a divisor of rows.  n is None with pre=NORM_NONE.  out may be x, out_n h."""
    where = "norm_residual"
    device = _device_of(where, x)
    if x.dim() != 2:
        raise ValueError(f"{where}: expected [rows, cols]")
    shape, kind, f32 = x.shape, x.dtype, _torch.float32
    rows, cols = shape
    col = (cols,)
    gate_rows = 0 if gate is None else gate.shape[0]
    y = _torch.empty_like(x) if out is None else out
    n = None
    if pre != NORM_NONE:
        n = _torch.empty_like(x) if out_n is None else out_n
    stats = _torch.empty((rows, 4), dtype=f32, device=x.device)
    check(lib().fdl_norm_residual(
        _given(where, "x", x, device, kind, shape), _given(where, "h", h, device, kind, shape),
        _given(where, "gate", gate, device, kind, (gate_rows, cols)), gate_rows, gate_act, post,
        _given(where, "post_gamma", post_gamma, device, f32, col), _given(where, "post_beta", post_beta, device, f32, col),
        pre, _given(where, "pre_gamma", pre_gamma, device, f32, col), _given(where, "pre_beta", pre_beta, device, f32, col),
        _given(where, "out", y, device, kind, shape), _given(where, "out_n", n, device, kind, shape), stats.data_ptr(),
        rows, cols, residual_scale, block_scale, eps, _dtype_code(where, x), _raw_stream(device)), "fdl_norm_residual")
    return y, n, stats


def norm_residual_backward(dy, dn, y, h, stats, post=NORM_RMS, pre=NORM_RMS, gate=None, gate_act=GATE_PLAIN,
                           post_gamma=None, post_beta=None, pre_gamma=None, residual_scale=1.0, block_scale=1.0,
                           want_post_beta=False, want_pre_beta=False):
    """Gradients of norm_residual as a dict: x, h, gate, post_gamma, post_beta, pre_gamma, pre_beta (None where there
    is nothing to learn).  dy or dn may be None."""
    where = "norm_residual_backward"
    device = _device_of(where, h)
    if h.dim() != 2:
        raise ValueError(f"{where}: expected [rows, cols]")
    shape, kind, f32 = h.shape, h.dtype, _torch.float32
    rows, cols = shape
    col = (cols,)
    gate_rows = 0 if gate is None else gate.shape[0]
    code = _dtype_code(where, h)
    like, place = _torch.empty_like, h.device
    bytes_ = lib().fdl_norm_residual_backward_scratch_bytes(rows, cols, gate_rows)
    scratch = _torch.empty((bytes_,), dtype=_torch.uint8, device=place)
    gx, gh, ggate = like(h), like(h), None if gate is None else like(gate)

    def beta_sum(wanted, gamma):
        if not wanted:
            return None
        return _torch.empty(col, dtype=f32, device=place) if gamma is None else like(gamma)

    sums = (None if post_gamma is None else like(post_gamma), beta_sum(want_post_beta, post_gamma),
            None if pre_gamma is None else like(pre_gamma), beta_sum(want_pre_beta, pre_gamma))
    check(lib().fdl_norm_residual_backward(
        _given(where, "dy", dy, device, kind, shape), _given(where, "dn", dn, device, kind, shape),
        _given(where, "y", y, device, kind, shape), _given(where, "h", h, device, kind, shape),
        _given(where, "stats", stats, device, f32, (rows, 4)), _given(where, "gate", gate, device, kind, (gate_rows, cols)),
        gate_rows, gate_act, post, _given(where, "post_gamma", post_gamma, device, f32, col),
        _given(where, "post_beta", post_beta, device, f32, col), pre,
        _given(where, "pre_gamma", pre_gamma, device, f32, col), gx.data_ptr(), gh.data_ptr(), _ptr(ggate), _ptr(sums[0]),
        _ptr(sums[1]), _ptr(sums[2]), _ptr(sums[3]), rows, cols, residual_scale, block_scale, code, scratch.data_ptr(),
        bytes_, _raw_stream(device)), "fdl_norm_residual_backward")
    return {"x": gx, "h": gh, "gate": ggate, "post_gamma": sums[0], "post_beta": sums[1], "pre_gamma": sums[2],
            "pre_beta": sums[3]}


def verify_draft(target, draft_tokens, accept_u, sample_u, draft=None, draft_len=None):
    """Drafted tokens against the target's probabilities: (tokens [batch, drafted + 1], accepted [batch]), int64.

    target [batch, drafted + 1, vocab], draft [batch, drafted, vocab] or None (a draft that is certain of its
    tokens), draft_tokens (int64) and accept_u [batch, drafted], sample_u [batch], draft_len (int64) [batch]."""
    where = "verify_draft"
    if target.dim() != 3 or draft_tokens.dim() != 2:
        raise ValueError(f"{where}: expected target [batch, drafted + 1, vocab] and draft_tokens [batch, drafted]")
    device = _device_of(where, target)
    kind, f32, i64 = target.dtype, _torch.float32, _torch.int64
    batch, drafted = draft_tokens.shape
    vocab = target.shape[2]
    target_batch, target_row, within = target.stride()
    draft_batch = draft_row = 0
    within_draft = 1
    if draft is not None:
        draft_batch, draft_row, within_draft = draft.stride()
    if vocab > 1 and not (within == within_draft == 1):
        raise ValueError(f"{where}: expected a contiguous last dimension")
    tokens = _torch.empty((batch, drafted + 1), dtype=i64, device=target.device)
    accepted = _torch.empty((batch,), dtype=i64, device=target.device)
    check(lib().fdl_verify_draft(
        _given(where, "target", target, device, kind, (batch, drafted + 1, vocab), contiguous=False), target_batch,
        target_row, _given(where, "draft", draft, device, kind, (batch, drafted, vocab), contiguous=False), draft_batch,
        draft_row, _dtype_code(where, target), _given(where, "draft_tokens", draft_tokens, device, i64, (batch, drafted)),
        _given(where, "draft_len", draft_len, device, i64, (batch,)),
        _given(where, "accept_u", accept_u, device, f32, (batch, drafted)),
        _given(where, "sample_u", sample_u, device, f32, (batch,)), batch, drafted, vocab, tokens.data_ptr(),
        accepted.data_ptr(), _raw_stream(device)), "fdl_verify_draft")
    return tokens, accepted


# ---- host-buffer entry points (torch CPU tensors, ideally pinned) ------------------------------


def host_binary(a, b, out, op):
    check(lib().fdl_host_binary_f32(_ptr(a), _ptr(b), _ptr(out), a.numel(), op), "fdl_host_binary_f32")
    return out


def host_unary(x, out, op, alpha=0.01):
    check(lib().fdl_host_unary_f32(_ptr(x), _ptr(out), x.numel(), op, alpha), "fdl_host_unary_f32")
    return out


def host_mul_add_relu(a, b, c, out):
    check(lib().fdl_host_mul_add_relu_f32(_ptr(a), _ptr(b), _ptr(c), _ptr(out), a.numel()),
          "fdl_host_mul_add_relu_f32")
    return out


def host_row_broadcast(a, row, out, op):
    rows, cols = a.shape
    check(lib().fdl_host_row_broadcast_f32(_ptr(a), _ptr(row), _ptr(out), rows, cols, op),
          "fdl_host_row_broadcast_f32")
    return out


def host_sum(x) -> float:
    res = C.c_double(0.0)
    check(lib().fdl_host_sum_f32(_ptr(x), x.numel(), C.byref(res)), "fdl_host_sum_f32")
    return res.value


def host_sweep(x, y, row, z, w) -> float:
    """z = x + y, w = x + row, returns sum(x); x, y, z, w are [rows, cols] host tensors."""
    rows, cols = x.shape
    res = C.c_double(0.0)
    check(lib().fdl_host_sweep_f32(_ptr(x), _ptr(y), _ptr(row), _ptr(z), _ptr(w), rows, cols, C.byref(res)),
          "fdl_host_sweep_f32")
    return res.value


# ---- cross-GPU exchange for the fused full sum ----------------------------------------------------


class Exchange:
    """Per-process context of fdl_sum_allreduce_f32.  `gather` is a callable that takes this
    rank's 64-byte handle and returns the list of all ranks' handles in rank order (for
    example a wrapper of torch.distributed.all_gather_object)."""

    def __init__(self, world: int, rank: int, gather):
        self.world, self.rank = world, rank
        ctx = C.c_void_p()
        check(lib().fdl_exchange_create(world, rank, C.byref(ctx)), "fdl_exchange_create")
        self.ctx = ctx
        buf = C.create_string_buffer(64)
        check(lib().fdl_exchange_local_handle(self.ctx, buf), "fdl_exchange_local_handle")
        handles = gather(buf.raw)
        if len(handles) != world or any(len(h) != 64 for h in handles):
            raise ValueError("exchange: expected one 64-byte handle per rank")
        check(lib().fdl_exchange_connect(self.ctx, b"".join(handles)), "fdl_exchange_connect")

    def sum(self, x, out32, out64):
        check(lib().fdl_sum_allreduce_f32(_ptr(x), x.numel(), _ptr(out32), _ptr(out64), self.ctx, None, 0,
                                          _stream()), "fdl_sum_allreduce_f32")

    def sum_start(self, x):
        """First half: the sum kernel sends this rank's partial to all ranks and does not wait."""
        check(lib().fdl_sum_allreduce_start_f32(_ptr(x), x.numel(), self.ctx, None, 0, _stream()),
              "fdl_sum_allreduce_start_f32")

    def sum_finish(self, out32, out64):
        """Second half: fold all ranks' partials (rank order) into the outputs."""
        check(lib().fdl_sum_allreduce_finish_f32(_ptr(out32), _ptr(out64), self.ctx, _stream()),
              "fdl_sum_allreduce_finish_f32")

    def reduce_cols(self, x2d, op, mean_divisor, out):
        rows, cols = x2d.shape
        check(lib().fdl_reduce_cols_allreduce_f32(_ptr(x2d), rows, cols, _ptr(out), op, float(mean_divisor),
                                                  self.ctx, None, 0, _stream()), "fdl_reduce_cols_allreduce_f32")
        return out

    def close(self):
        if self.ctx:
            lib().fdl_exchange_destroy(self.ctx)
            self.ctx = None
