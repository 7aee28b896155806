"""Dense feed-forward operators on top of the C ABI (include/zc_ffn.h): microscaled 4-bit matrices and the gated block in 16 bits with
its gradient - the shared or dense form of the block whose routed form is ``zerocool_b200.moe``.

    w = mx4_quantize(weight)                  # once: codes and scales, 17/32 byte a value
    h = mx4_gated(x, gate, up)                # silu(x gate^T) * (x up^T), one kernel
    y = mx4_linear(h, down)                   # x of a product: plain (quantised on the way) or an Mx4

    h, g, u = gated_forward(x, gate, up, save=True)
    dx, dgate, dup = gated_backward(dh, x, gate, up, g, u)

Calls run on the tensors' device and torch's current stream of it, allocate results and scratch with torch and may be captured into a
CUDA graph, the first call of a process too. Nothing here has a CPU path, and autograd does not see these calls: a block or product of tensors that
require gradients is refused where gradients are recorded, as its result would silently have none (call it under ``torch.no_grad()``, or pass
``x.detach()``). Errors are those of ``zerocool_b200.moe``: ``ValueError`` for arguments, ``RuntimeError`` for the device.
"""
import ctypes

import torch

from . import moe
from .records import BF16, F16, F32

EXPORTS = ["zc_mx4_scale_bytes", "zc_mx4_quantize", "zc_mx4_dequantize", "zc_mx4_tile_scales", "zc_mx4_linear", "zc_mx4_gated",
           "zc_gated_forward", "zc_gated_backward", "zc_ffn_status", "zc_ffn_wait_limit"]

_lib = None
# torch's handle of the current stream without a Stream object around it (2 us less a call); absent from builds without CUDA.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def load_library():
    """The library of ``zerocool_b200.moe`` with the prototypes of include/zc_ffn.h."""
    global _lib
    if _lib is None:
        lib = moe.load_library()
        vp, u32, u64, i32 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int
        lib.zc_mx4_scale_bytes.argtypes = [u32, u32, ctypes.POINTER(u64)]
        lib.zc_mx4_quantize.argtypes = [vp, i32, u32, u32, u64, vp, vp, vp]
        lib.zc_mx4_dequantize.argtypes = [vp, vp, u32, u32, vp, i32, u64, vp]
        lib.zc_mx4_tile_scales.argtypes = [vp, u32, u32, vp, vp]
        lib.zc_mx4_linear.argtypes = [vp, i32, u64, vp, vp, u32, u32, vp, vp, u32, vp, i32, u64, vp]
        lib.zc_mx4_gated.argtypes = [vp, i32, u64, vp, vp, u32, u32, vp, vp, vp, vp, u32, vp, i32, u64, vp]
        lib.zc_gated_forward.argtypes = [vp, u64, vp, vp, i32, u32, u32, u32, vp, vp, vp, i32, vp]
        lib.zc_gated_backward.argtypes = [vp, u64, vp, u64, vp, vp, vp, vp, i32, i32, u32, u32, u32, vp, vp, vp, vp, vp, vp]
        lib.zc_ffn_status.argtypes = [vp, ctypes.POINTER(u32)]
        lib.zc_ffn_wait_limit.argtypes = [u32, ctypes.POINTER(u32)]
        _lib = lib
    return _lib


CODES = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}


def _code(dtype, sixteen=False):
    if dtype not in CODES or (sixteen and dtype == torch.float32):
        raise ValueError(f"dtype must be {'bfloat16 or float16' if sixteen else 'bfloat16, float16 or float32'}, not {dtype}")
    return CODES[dtype]


def _matrix(name, t, shape=None, dtype=None, contiguous=False):
    """Checks a matrix operand; -> its row stride in elements."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError(f"{name} must be a matrix")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    rows, cols = t.shape
    if t.is_contiguous():
        return cols
    if contiguous:
        raise ValueError(f"{name} must be contiguous")
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
        raise ValueError(f"{name} must have consecutive columns and rows that do not overlap")
    return t.stride(0) if rows > 1 else cols


def _whole(name, t, shape, dtype, device):
    """Checks a contiguous matrix of this shape, type and device: all at once, and one by one where that fails."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device and t.is_contiguous()):
        _matrix(name, t, shape, dtype, contiguous=True)
        _same_device(device, **{name: t})


def _unrecorded():
    """For operands that require gradients."""
    if torch.is_grad_enabled():
        raise ValueError("autograd does not see this call: its result would not have the gradient that its operands require (torch.no_grad(), or detach them)")


def _tensor(name, t):
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError(f"{name} must be a matrix")


def _mx4(name, q):
    if not isinstance(q, Mx4):
        raise ValueError(f"{name} must be an Mx4 (mx4_quantize)")


def _same_device(device, **others):
    for name, t in others.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _call(device, name, *args):
    """One library call on the device's current stream (its last argument), with that device current."""
    lib = _lib or load_library()
    stream = _raw_stream(device.index) if _raw_stream else torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        rc = getattr(lib, name)(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = getattr(lib, name)(*args, stream)
    if rc != moe.ZC_OK:
        moe._raise(rc, lib.zc_last_error())


def _scale_bytes(rows, cols):
    return -(-rows // 128) * -(-cols // 128) * 512


def _out(out, rows, cols, dtype, device, name="out"):
    """The output matrix and its row stride."""
    if out is None:
        return torch.empty((rows, cols), dtype=dtype, device=device), cols
    ld = _matrix(name, out, (rows, cols), dtype)
    _same_device(device, **{name: out})
    return out, ld


class Mx4:
    """A microscaled matrix [rows, cols]: codes uint8 [rows, cols / 2] and scales uint8 [ceil(rows / 128) ceil(cols / 128) 512] in the
    tile layout of include/zc_ffn.h. Holds the tensors; copies nothing."""

    def __init__(self, codes, scales):
        _tensor("codes", codes)
        if not isinstance(scales, torch.Tensor):
            raise ValueError("scales must be a tensor")
        if codes.dtype != torch.uint8 or not codes.is_contiguous() or codes.shape[1] % 16 or not codes.shape[1]:
            raise ValueError("codes must be contiguous uint8 [rows, cols / 2], cols a multiple of 32")
        if scales.dtype != torch.uint8 or not scales.is_contiguous() or scales.device != codes.device or \
                scales.numel() != _scale_bytes(codes.shape[0], codes.shape[1] * 2):
            raise ValueError("scales must be contiguous uint8 of the codes' device, 512 for each 128 rows x 128 columns")
        if not codes.is_cuda:
            raise ValueError("codes must be on a CUDA device")
        self.codes, self.scales = codes, scales

    @property
    def rows(self):
        return self.codes.shape[0]

    @property
    def cols(self):
        return self.codes.shape[1] * 2

    @property
    def device(self):
        return self.codes.device

    @staticmethod
    def empty(rows, cols, device):
        """A matrix whose values are yet to be written (mx4_quantize(..., out=))."""
        if not isinstance(rows, int) or not isinstance(cols, int) or rows < 0 or cols <= 0 or cols % 32:
            raise ValueError("rows and columns must be whole numbers, columns a multiple of 32")
        q = object.__new__(Mx4)          # nothing to check
        q.codes = torch.empty((rows, cols // 2), dtype=torch.uint8, device=device)
        if not q.codes.is_cuda:
            raise ValueError("the device must be a CUDA device")
        q.scales = q.codes.new_empty(_scale_bytes(rows, cols))
        return q


def mx4_quantize(x, out=None):
    """x [rows, cols] (bfloat16, float16 or float32, cols a multiple of 32) -> Mx4; ``out``: an Mx4 of that shape to write."""
    ld = _matrix("x", x)
    rows, cols = x.shape
    if out is None:
        out = Mx4.empty(rows, cols, x.device)
    else:
        _mx4("out", out)
        if (out.rows, out.cols) != (rows, cols):
            raise ValueError(f"out must be [{rows}, {cols}]")
        _same_device(x.device, out=out)
    _call(x.device, "zc_mx4_quantize", x.data_ptr(), _code(x.dtype), rows, cols, ld, out.codes.data_ptr(), out.scales.data_ptr())
    return out


def mx4_dequantize(q, dtype=None, out=None):
    """The values of an Mx4 (default bfloat16, which holds each of them exactly)."""
    _mx4("q", q)
    dtype = getattr(out, "dtype", None) if dtype is None and out is not None else dtype or torch.bfloat16
    code = _code(dtype)
    out, ld = _out(out, q.rows, q.cols, dtype, q.device)
    _call(q.device, "zc_mx4_dequantize", q.codes.data_ptr(), q.scales.data_ptr(), q.rows, q.cols, out.data_ptr(), code, ld)
    return out


def mx4_from_rows(codes, scales):
    """A checkpoint's codes [rows, cols / 2] and row-major scales [rows, cols / 32] (both uint8) -> Mx4 (the codes are not copied)."""
    _tensor("codes", codes)
    _tensor("scales", scales)
    if codes.dtype != torch.uint8:
        raise ValueError("codes must be uint8 [rows, cols / 2]")
    if scales.dtype != torch.uint8 or not scales.is_contiguous() or tuple(scales.shape) != (codes.shape[0], codes.shape[1] // 16):
        raise ValueError("scales must be contiguous uint8 [rows, cols / 32]")
    q = Mx4(codes, torch.empty(_scale_bytes(codes.shape[0], codes.shape[1] * 2), dtype=torch.uint8, device=codes.device))
    _same_device(codes.device, scales=scales)
    _call(codes.device, "zc_mx4_tile_scales", scales.data_ptr(), q.rows, q.cols, q.scales.data_ptr())
    return q


def _mx4_product(entry, x, weights, out_dtype, out):
    for w in weights:
        if not isinstance(w, Mx4):
            raise ValueError("the weights must be Mx4 (mx4_quantize)")
    w = weights[0]
    device, cols, rows = w.device, w.cols, w.rows
    for other in weights[1:]:
        if (other.rows, other.cols) != (rows, cols):
            raise ValueError(f"the weights differ in shape: [{rows}, {cols}] and [{other.rows}, {other.cols}]")
    if isinstance(x, Mx4):
        tokens, xcols, plain = x.rows, x.cols, (None, F32, 0)
        codes, scales = x.codes.data_ptr(), x.scales.data_ptr()
    else:
        ld = _matrix("x", x)
        if x.requires_grad:
            _unrecorded()
        (tokens, xcols), plain = x.shape, (x.data_ptr(), _code(x.dtype), ld)
        scratch = torch.empty(tokens * cols // 2 + _scale_bytes(tokens, cols), dtype=torch.uint8, device=device)      # codes, then scales
        codes = scratch.data_ptr()
        scales = codes + tokens * cols // 2
    if xcols != cols:
        raise ValueError(f"x has {xcols} columns, the weights {cols}")
    _same_device(device, x=x, weights=weights[-1])
    out_dtype = getattr(out, "dtype", None) if out_dtype is None and out is not None else out_dtype or torch.bfloat16
    code = _code(out_dtype)
    out, out_ld = _out(out, tokens, rows, out_dtype, device)
    pointers = [p for m in weights for p in (m.codes.data_ptr(), m.scales.data_ptr())]
    _call(device, entry, *plain, codes, scales, tokens, cols, *pointers, rows, out.data_ptr(), code, out_ld)
    return out


def mx4_linear(x, w, out_dtype=None, out=None):
    """x w^T [tokens, w.rows] in out_dtype (default bfloat16): x an Mx4 or a plain matrix [tokens, w.cols], w an Mx4."""
    return _mx4_product("zc_mx4_linear", x, [w], out_dtype, out)


def mx4_gated(x, gate, up, out_dtype=None, out=None):
    """silu(x gate^T) * (x up^T) [tokens, ffn] in out_dtype (default bfloat16): x as in mx4_linear, gate and up Mx4 [ffn, cols]."""
    return _mx4_product("zc_mx4_gated", x, [gate, up], out_dtype, out)


def gated_forward(x, gate, up, save=False, save_dtype=torch.float32, out=None):
    """silu(x gate^T) * (x up^T): x [tokens, hidden], gate and up [ffn, hidden], one of bfloat16 and float16; -> h [tokens, ffn], and
    with ``save`` (h, g, u): the two products as gated_backward wants them, in float32, or in the operands' dtype for half the memory and
    two more roundings in the gradients."""
    code = _code(getattr(x, "dtype", None), sixteen=True)
    ld = _matrix("x", x)
    _tensor("gate", gate)
    (tokens, hidden), ffn = x.shape, gate.shape[0]
    dtype, device = x.dtype, x.device
    _whole("gate", gate, (ffn, hidden), dtype, device)
    _whole("up", up, (ffn, hidden), dtype, device)
    if x.requires_grad or gate.requires_grad or up.requires_grad:
        _unrecorded()
    if out is None:
        out = x.new_empty((tokens, ffn))
    else:
        _whole("out", out, (tokens, ffn), dtype, device)
    g, u, saved = None, None, code
    if save:
        if save_dtype not in (torch.float32, x.dtype):
            raise ValueError(f"save_dtype must be float32 or {x.dtype}, not {save_dtype}")
        g, u, saved = torch.empty_like(out, dtype=save_dtype), torch.empty_like(out, dtype=save_dtype), CODES[save_dtype]
    _call(device, "zc_gated_forward", x.data_ptr(), ld, gate.data_ptr(), up.data_ptr(), code, tokens, hidden, ffn, out.data_ptr(),
          g.data_ptr() if save else None, u.data_ptr() if save else None, saved)
    return (out, g, u) if save else out


def gated_backward(dh, x, gate, up, g, u, input_grad=True, weight_grads=True):
    """The gradient of gated_forward -> (dx, dgate, dup) in the operands' dtype (None for what is not asked for)."""
    code = _code(getattr(x, "dtype", None), sixteen=True)
    x_ld = _matrix("x", x)
    _tensor("gate", gate)
    (tokens, hidden), ffn = x.shape, gate.shape[0]
    dtype, device = x.dtype, x.device
    _whole("gate", gate, (ffn, hidden), dtype, device)
    _whole("up", up, (ffn, hidden), dtype, device)
    dh_ld = _matrix("dh", dh, (tokens, ffn), dtype)
    _same_device(device, dh=dh)
    saved = torch.float32 if getattr(g, "dtype", None) == torch.float32 else dtype
    _whole("g", g, (tokens, ffn), saved, device)
    _whole("u", u, (tokens, ffn), saved, device)
    if not input_grad and not weight_grads:
        return None, None, None
    scratch = x.new_empty((2, tokens, ffn))      # dg, du
    dx = x.new_empty((tokens, hidden)) if input_grad else None
    dgate, dup = (torch.empty_like(gate), torch.empty_like(up)) if weight_grads else (None, None)
    pointer = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _call(device, "zc_gated_backward", dh.data_ptr(), dh_ld, x.data_ptr(), x_ld, gate.data_ptr(), up.data_ptr(), g.data_ptr(), u.data_ptr(), CODES[saved], code,
          tokens, hidden, ffn, scratch.data_ptr(), scratch.data_ptr() + tokens * ffn * 2, pointer(dx), pointer(dgate), pointer(dup))
    return dx, dgate, dup


def status(device=None):
    """Waits for the device's current stream and returns (then clears) the device's status word of these operators, the same for all of its streams."""
    word = ctypes.c_uint32()
    lib = load_library()
    with torch.cuda.device(device):
        rc = lib.zc_ffn_status(torch.cuda.current_stream().cuda_stream, ctypes.byref(word))
    if rc != moe.ZC_OK:
        moe._raise(rc, lib.zc_last_error())
    return word.value


WAIT_POLLS = 1 << 20


def wait_limit(polls=WAIT_POLLS):
    """Sets how often a wait inside the products' kernels polls before it gives up (zc_ffn_wait_limit); -> the limit so far."""
    if isinstance(polls, bool) or not isinstance(polls, int) or not 0 <= polls <= 1 << 27:
        raise ValueError("polls must be a whole number up to 2^27")
    before = ctypes.c_uint32()
    load_library().zc_ffn_wait_limit(polls, ctypes.byref(before))
    return before.value
