"""Python front-end of the 4-bit matrix-vector products (``csrc/tk_gemv_w4.hip``).

``gemv_w4(x, codes, scales, zeros)`` multiplies 1 to 64 rows of ``x`` -- one token, or a
decode batch -- with a weight of 4-bit codes and a scale (and a zero) per group of columns,
``w[n][k] = scales[n][k // group] * (codes[n][k] - zeros[n][k // group])``.  Like
``gemm.gemm_bt`` it takes torch tensors on the GPU and queues its work on torch's current
stream of that device.  ``quantize_w4``, ``pack_w4`` and ``dequantize_w4`` make such weights
and undo them, on any device.
"""

import ctypes
import math
import struct
from typing import Any, Optional, Tuple

from .native import NativeUnavailable, load

MAX_ROWS = 64
MAX_OUT = 1 << 24
MAX_IN = 1 << 20
SYMMETRIC_ZERO = 8  # the zero of weights without zeros


class GemvError(RuntimeError):
    pass


# struct tkv_args of csrc/tk_gemv_w4.hip: dev f16 m n k group splits, ldx ldy, x codes scales zeros
# y part stream
_ARGS = struct.Struct("@7i2q7P")

_loaded = None


def _lib():
    global _loaded
    if _loaded is None:
        from .native import require_torch_first

        require_torch_first()
        lib = load("libtk_gemv.so")
        lib.tkv_last_error.restype = ctypes.c_char_p
        lib.tkv_gemv_w4.argtypes = [ctypes.c_char_p]
        if lib.tkv_args_size() != _ARGS.size:
            raise NativeUnavailable("libtk_gemv.so does not match ops/gemv.py: run `python -m triton_kubernetes_amd.ops.build`")
        _loaded = lib
    return _loaded


def _check_weight(codes, scales, zeros) -> Tuple[int, int, int]:
    """``(n, k, group)`` of a packed weight."""
    import torch

    shape, by = codes.shape, scales.shape
    if codes.dtype is not torch.uint8 or len(shape) != 2 or len(by) != 2 or by[0] != shape[0]:
        raise GemvError(f"wants codes uint8 [N, K/2] and scales [N, K/group], not {codes.dtype} {list(codes.shape)} "
                        f"and {list(scales.shape)}")
    n, half = shape
    k, groups = half * 2, by[1]
    if not groups or not k or k % groups or k // groups % 32:
        raise GemvError(f"{groups} groups do not divide {k} columns into groups of a multiple of 32")
    if zeros is not None and (zeros.dtype is not torch.uint8 or zeros.shape != by):
        raise GemvError(f"wants zeros uint8 {list(scales.shape)}, not {zeros.dtype} {list(zeros.shape)}")
    return n, k, k // groups


def splits(m: int, n: int, k: int) -> int:
    """How the product is run: 0, each row of ``x`` by itself, or into how many parts ``k`` is split.

    A row by itself is one launch and no join, and small weights come out of the cache for every
    row (4 x 1024 x 4096: 5.7 us, 6.9 together; 8 rows 7.2 and 7.0; 2 x 4096 x 4096 7.9 and 7.7,
    4 rows 10.3 and 7.9; 64 x 1024 x 512 6.2 and 9.2).  Together a workgroup takes 128 rows of the
    weight (256 for more than 16 rows of ``x``), and one for each of the 256 compute units is best
    (64 rows of ``x``, 16384 x 16384: 64 us; 99 with 128 of them, 75 with 512, whose sums cost more
    to join); a part has at least 2 chunks of 128 columns, a stage."""
    if m == 1 or m * n * k < 1 << 25:
        return 0
    blocks = -(-n // (128 if m <= 16 else 256))
    chunks = -(-k // 128)
    want = max(1, min(256 // blocks, chunks // 2, 64))
    per = _up(-(-chunks // want), 2)
    return -(-chunks // per)  # no part is empty


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def _overlap(a, b) -> bool:
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.element_size() * (
        1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))) for t in (a, b))
    return a0 < b1 and b0 < a1


def _tangents(*tensors) -> bool:
    """Whether one of them carries a forward-mode derivative (no_grad says nothing of these)."""
    from torch.autograd import forward_ad

    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def gemv_w4(x, codes, scales, zeros=None, *, out=None):
    """``x @ w.T`` for ``x [..., K]`` of at most 64 rows, bf16 or fp16, of any strides.

    ``codes`` is uint8 ``[N, K/2]``, two codes to a byte, the lower half first; ``scales``
    ``[N, K/group]`` has ``x``'s type, ``zeros`` (uint8, the same shape) may be left out for
    symmetric weights, whose zero is 8.  The weight's tensors are contiguous; ``group`` is a
    multiple of 32.  Sums are fp32 and rounded once; they are of ``(16 + code) * x``, so an
    infinite ``x`` gives NaN.  The result (``out``, if given: contiguous, ``[..., N]``, changed
    in place as torch counts it) has ``x``'s type.  It is for serving: it has no gradient, and an ``x`` that wants one,
    or that has a forward-mode tangent, is refused."""
    import torch

    dtype = x.dtype
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or scales.dtype is not dtype:
        raise GemvError(f"gemv_w4 wants x and scales both bf16 or both fp16, not {x.dtype} and {scales.dtype}")
    n, k, group = _check_weight(codes, scales, zeros)
    shape = x.shape
    if len(shape) < 1 or shape[-1] != k:
        raise GemvError(f"x {list(shape)} does not go with {k} columns")
    if n > MAX_OUT or k > MAX_IN:
        raise GemvError(f"a weight of {n} x {k} (at most {MAX_OUT} x {MAX_IN})")
    dev = x.get_device()
    if dev < 0 or codes.get_device() != dev or scales.get_device() != dev or (zeros is not None and zeros.get_device() != dev):
        raise GemvError("gemv_w4 wants CUDA tensors on one device")
    at = codes.data_ptr()
    if at % 16 or not (codes.is_contiguous() and scales.is_contiguous() and (zeros is None or zeros.is_contiguous())):
        raise GemvError("gemv_w4 wants a contiguous weight, its codes 16-byte aligned")
    if (x.requires_grad or scales.requires_grad) and torch.is_grad_enabled():
        raise GemvError("gemv_w4 has no gradient: call it under torch.no_grad()")
    if torch.autograd.forward_ad._current_level >= 0 and _tangents(x, scales, out):  # (0.1 us, 0.9 always)
        raise GemvError("gemv_w4 has no gradient: a tensor with a tangent has to be unpacked first")
    flat = len(shape) == 2
    m = shape[0] if flat else x.numel() // k
    if m > MAX_ROWS:
        raise GemvError(f"{m} rows of x (at most {MAX_ROWS}): dequantize_w4 and a matrix product serve more")
    if out is None:
        out = x.new_empty((m, n) if flat else (*shape[:-1], n))
    elif out.shape != (*shape[:-1], n) or out.dtype is not dtype or out.device != x.device or not out.is_contiguous():
        raise GemvError(f"out must be contiguous {dtype} {[*shape[:-1], n]} on x's device")
    elif any(_overlap(out, t) for t in (x, codes, scales, zeros) if t is not None):
        raise GemvError("out must not share memory with x or the weight")
    elif out.requires_grad and torch.is_grad_enabled():
        raise GemvError("gemv_w4 has no gradient: call it under torch.no_grad()")
    elif not out.is_inference():
        torch.autograd.graph.increment_version(out)  # the kernel writes it behind torch's back
    if m == 0 or n == 0:
        return out
    if not flat:
        x = x.reshape(m, k)
    ldx, step = x.stride()
    if m == 1:
        ldx = k
    from_x = x.data_ptr()
    if step != 1 or ldx < k or ldx % 8 or from_x % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        ldx, from_x = k, x.data_ptr()
    parts = splits(m, n, k)
    room = x.new_empty((parts, m, n), dtype=torch.float32) if parts > 1 else None
    lib = _loaded or _lib()
    if lib.tkv_gemv_w4(_ARGS.pack(dev, dtype is torch.float16, m, n, k, group, parts, ldx, n, from_x, at, scales.data_ptr(),
                                  0 if zeros is None else zeros.data_ptr(), out.data_ptr(),
                                  0 if room is None else room.data_ptr(), torch._C._cuda_getCurrentRawStream(dev))) != 0:
        raise GemvError(lib.tkv_last_error().decode())
    return out


def pack_w4(codes):
    """Codes 0 to 15, uint8 ``[N, K]``, as ``[N, K/2]``: two to a byte, the lower half first."""
    import torch

    if codes.dtype != torch.uint8 or codes.dim() != 2 or codes.shape[1] % 2:
        raise GemvError(f"pack_w4 wants uint8 [N, K] with an even K, not {codes.dtype} {list(codes.shape)}")
    if codes.numel() and int(codes.max()) > 15:
        raise GemvError("pack_w4 wants codes 0 to 15")
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def quantize_w4(w, group: int = 128, symmetric: bool = True) -> Tuple[Any, Any, Optional[Any]]:
    """``(codes, scales, zeros)`` of a bf16 or fp16 weight ``[N, K]``, each value to the code
    nearest to it; ``zeros`` is None for a symmetric weight.  A symmetric group's scale is its
    largest magnitude / 7; else scale and zero span the group's values (and 0) with 15 steps."""
    import torch

    if w.dtype not in (torch.bfloat16, torch.float16) or w.dim() != 2:
        raise GemvError(f"quantize_w4 wants bf16 or fp16 [N, K], not {w.dtype} {list(w.shape)}")
    n, k = w.shape
    if group < 32 or group % 32 or k < group or k % group:
        raise GemvError(f"a group of {group} must be a multiple of 32 that divides {k} columns")
    v = w.detach().float().reshape(n, k // group, group)
    if not bool(torch.isfinite(v).all()):
        raise GemvError("quantize_w4 wants finite weights")
    if symmetric:
        scales = (v.abs().amax(2) / 7).to(w.dtype)
        zeros = None
    else:
        lo, hi = v.amin(2).clamp_max(0), v.amax(2).clamp_min(0)
        if not bool(torch.isfinite(hi - lo).all()):
            raise GemvError("quantize_w4 wants groups whose span is an fp32 number")
        scales = ((hi - lo) / 15).to(w.dtype)
    # codes go by the rounded scale; a scale of 0 (a group of zeros, or too small for the type) has code = zero
    step = scales.float()
    step = torch.where(step > 0, step, math.inf)
    if not symmetric:
        zeros = (-lo / step).round().clamp(0, 15).to(torch.uint8)
    zero = float(SYMMETRIC_ZERO) if zeros is None else zeros.float()[:, :, None]
    codes = (v / step[:, :, None] + zero).round().clamp(0, 15).to(torch.uint8)
    return pack_w4(codes.reshape(n, k)), scales, zeros


def dequantize_w4(codes, scales, zeros=None):
    """The weight ``[N, K]`` in fp32."""
    import torch

    n, k, group = _check_weight(codes, scales, zeros)
    c = torch.stack((codes & 15, codes >> 4), 2).reshape(n, k // group, group).float()
    zero = float(SYMMETRIC_ZERO) if zeros is None else zeros.float()[:, :, None]
    return ((c - zero) * scales.float()[:, :, None]).reshape(n, k)
