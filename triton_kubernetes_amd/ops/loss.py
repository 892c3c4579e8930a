"""Python front-end of the output head's losses (``csrc/tk_loss.hip``).

``linear_cross_entropy(x, w, target)`` is the softmax cross entropy of the logits ``x @ w.T``,
and ``linear_distill(x, w, ids, logits)`` their divergence from a teacher's top logits; both
with their gradients (torch autograd), and without the ``[tokens, vocabulary]`` logits ever
being stored: the forward pass keeps a few numbers a token, and the backward pass computes
the logits again, a piece of the vocabulary at a time.  Like ``gemm.gemm_bt`` they take torch
tensors on the GPU and queue their work on torch's current stream of that device; nothing
waits for it here, and both directions can be captured into a graph.
"""

import ctypes
from typing import Any, Tuple

from .native import NativeUnavailable, load

TILE = 256  # vocabulary entries and tokens of a tile
DL_BYTES = 512 << 20  # the backward pass' 16-bit derivative of the logits, per piece
DX_BYTES = 512 << 20  # fp32 partial sums of x's gradient, over the splits
MAX_TARGETS = 1024  # ids of a token's list
MAX_TOKENS = 1 << 20
MAX_WIDTH = 1 << 16
MAX_VOCAB = 1 << 24
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


class LossError(RuntimeError):
    pass


_LL, _I, _F, _P = ctypes.c_longlong, ctypes.c_int, ctypes.c_float, ctypes.c_void_p


class _Args(ctypes.Structure):
    """``struct tkl_args`` of ``csrc/tk_loss.hip``."""

    _fields_ = ([(f, _LL) for f in ("n", "d", "v", "k", "ldx", "ldw", "ldg", "ignore", "piece", "splits")]
                + [(f, _I) for f in ("dev", "f16", "distill", "reduction")] + [("temperature", _F), ("want", _I)]
                + [(f, _P) for f in ("x", "w", "ids", "teacher", "grad", "loss", "xc", "lse", "zk", "p", "rowloss",
                                     "rowmap", "posof", "count", "flag", "part", "wc", "dl", "dxpart", "factor", "dx",
                                     "dw", "stream")])


_loaded = None


def _lib():
    global _loaded
    if _loaded is None:
        lib = load("libtk_loss.so")
        lib.tkl_last_error.restype = ctypes.c_char_p
        lib.tkl_forward.argtypes = [ctypes.POINTER(_Args)]
        lib.tkl_backward.argtypes = [ctypes.POINTER(_Args)]
        if lib.tkl_args_size() != ctypes.sizeof(_Args):
            raise NativeUnavailable("libtk_loss.so does not match ops/loss.py: run `python -m triton_kubernetes_amd.ops.build`")
        _loaded = lib
    return _loaded


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def pieces(n: int, v: int) -> int:
    """Vocabulary entries of a piece of the backward pass: as many as keep the derivative of
    ``n`` tokens' logits under ``DL_BYTES``, spread evenly, in whole tiles."""
    most = max(TILE, DL_BYTES // (2 * n) // TILE * TILE)
    return _up(-(-v // -(-v // most)), TILE)


def splits(n: int, d: int, piece: int) -> int:
    """Into how many parts the vocabulary is split for x's gradient: enough tiles for 256
    compute units, at least 512 entries a part, and no more than ``DX_BYTES`` of sums."""
    tiles = -(-n // TILE) * -(-d // TILE)
    return max(1, min(512 // tiles, piece // 512, DX_BYTES // (4 * n * _up(d, 64))))


def _padded_weight(w) -> bool:
    """Whether the kernels need a copy of ``w`` with padded rows."""
    d = w.shape[1]
    return bool(d % 8 or w.stride(0) % 8 or w.data_ptr() % 16)


def _plain(w):
    """``w`` with a row stride that the kernels take."""
    return w if w.stride(1) == 1 and w.shape[1] <= w.stride(0) <= 1 << 21 else w.contiguous()


class _Kept:
    """Sizes, settings and the addresses of what the forward pass keeps for the backward pass."""

    __slots__ = ("n", "d", "v", "k", "distill", "reduction", "temperature", "ignore")

    def fields(self, a: _Args, slab) -> None:
        """The addresses within ``slab``, one fp32 tensor that holds them all."""
        at, n, k = slab.data_ptr(), self.n, self.k
        for name, count in (("lse", n), ("rowloss", n), ("rowmap", n), ("posof", n), ("count", 1), ("zk", n * k),
                            ("p", n * k if self.distill else 0), ("flag", n if self.distill else 0)):
            setattr(a, name, at)
            at += 4 * count

    def words(self) -> int:
        return 4 * self.n + 1 + self.n * self.k + (self.n * (self.k + 1) if self.distill else 0)

    def args(self, device, f16: bool, slab) -> _Args:
        import torch

        a = _Args(n=self.n, d=self.d, v=self.v, k=self.k, ignore=self.ignore, distill=self.distill,
                  reduction=self.reduction, temperature=self.temperature, f16=f16, dev=device.index,
                  stream=torch.cuda.current_stream(device).cuda_stream)
        self.fields(a, slab)
        return a


_function = None


def _autograd():
    """The autograd function (torch is imported on first use)."""
    global _function
    if _function is not None:
        return _function
    import torch

    class HeadLoss(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, ids, teacher, kept):
            dev = x.device
            f16 = x.dtype == torch.float16
            lead = x.shape[:-1]
            ctx.kept, ctx.lead = kept, lead
            loss = torch.empty(lead if kept.reduction == 0 else (), dtype=torch.float32, device=dev)
            if kept.n == 0 or kept.k == 0:  # nothing has a loss
                ctx.save_for_backward(x, w)
                return loss.zero_()
            x = x.reshape(-1, kept.d)
            if x.stride(1) != 1:
                x = x.contiguous()
            plain = _plain(w)
            dp = _up(kept.d, 64)
            xc = torch.empty((kept.n, dp), dtype=x.dtype, device=dev)
            slab = torch.empty(kept.words(), dtype=torch.float32, device=dev)
            part = torch.empty(4 * -(-kept.v // TILE) * kept.n, dtype=torch.float32, device=dev)
            a = kept.args(dev, f16, slab)
            wc = torch.empty((kept.v, dp), dtype=w.dtype, device=dev) if _padded_weight(plain) else None
            a.x, a.ldx, a.w, a.ldw, a.ids = x.data_ptr(), x.stride(0), plain.data_ptr(), plain.stride(0), ids.data_ptr()
            a.teacher = teacher.data_ptr() if teacher is not None else None
            a.wc = wc.data_ptr() if wc is not None else None
            a.loss, a.xc, a.part = loss.data_ptr(), xc.data_ptr(), part.data_ptr()
            if _lib().tkl_forward(ctypes.byref(a)) != 0:
                raise LossError(_lib().tkl_last_error().decode())
            ctx.save_for_backward(w, ids, xc, slab)
            return loss

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            kept = ctx.kept
            want = (1 if ctx.needs_input_grad[0] else 0) | (2 if ctx.needs_input_grad[1] else 0)
            if kept.n == 0 or kept.k == 0:
                x, w = ctx.saved_tensors
                return (torch.zeros_like(x) if want & 1 else None, torch.zeros_like(w) if want & 2 else None, None, None,
                        None)
            w, ids, xc, slab = ctx.saved_tensors
            dev = xc.device
            if kept.reduction == 0:
                grad = grad.reshape(-1)
            grad = grad.float()
            plain = _plain(w)
            dp = _up(kept.d, 64)
            a = kept.args(dev, xc.dtype == torch.float16, slab)
            a.want, a.piece = want, pieces(kept.n, kept.v)
            a.splits = splits(kept.n, kept.d, a.piece)
            a.grad, a.ldg = grad.data_ptr(), grad.stride(0) if kept.reduction == 0 else 0
            a.w, a.ldw, a.ids, a.xc = plain.data_ptr(), plain.stride(0), ids.data_ptr(), xc.data_ptr()
            wc = torch.empty((kept.v, dp), dtype=w.dtype, device=dev) if _padded_weight(plain) else None
            a.wc = wc.data_ptr() if wc is not None else None
            dl = torch.empty((kept.n, a.piece), dtype=xc.dtype, device=dev)
            factor = torch.empty(kept.n + 1, dtype=torch.float32, device=dev)
            a.dl, a.factor = dl.data_ptr(), factor.data_ptr()
            dx = dw = None
            if want & 1:
                dxpart = torch.empty((a.splits, kept.n, dp), dtype=torch.float32, device=dev)
                dx = torch.empty((kept.n, kept.d), dtype=xc.dtype, device=dev)
                a.dxpart, a.dx = dxpart.data_ptr(), dx.data_ptr()
            if want & 2:
                dw = torch.empty((kept.v, kept.d), dtype=xc.dtype, device=dev)
                a.dw = dw.data_ptr()
            if want and _lib().tkl_backward(ctypes.byref(a)) != 0:
                raise LossError(_lib().tkl_last_error().decode())
            return None if dx is None else dx.view(*ctx.lead, kept.d), dw, None, None, None

    _function = HeadLoss
    return _function


def _check(what: str, x, w, reduction: str) -> Tuple[Any, _Kept]:
    import torch

    from .native import require_torch_first

    require_torch_first()
    if x.dtype not in (torch.bfloat16, torch.float16) or w.dtype != x.dtype:
        raise LossError(f"{what} wants x and w both bf16 or both fp16, not {x.dtype} and {w.dtype}")
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise LossError(f"{what} wants x [..., D] and w [V, D], not {list(x.shape)} and {list(w.shape)}")
    if not (x.is_cuda and w.is_cuda) or x.device != w.device:
        raise LossError(f"{what} wants CUDA tensors on one device, not {x.device} and {w.device}")
    if reduction not in REDUCTIONS:
        raise LossError(f"unknown reduction '{reduction}' ({' | '.join(REDUCTIONS)})")
    kept = _Kept()
    kept.v, kept.d = w.shape
    kept.n = x.numel() // kept.d if kept.d else 0
    kept.reduction = REDUCTIONS[reduction]
    if not (1 <= kept.d <= MAX_WIDTH and 1 <= kept.v <= MAX_VOCAB and kept.n <= MAX_TOKENS):
        raise LossError(f"{what}: {kept.n} tokens of width {kept.d} over {kept.v} entries (at most {MAX_TOKENS}, "
                        f"{MAX_WIDTH}, {MAX_VOCAB})")
    return x, kept


_INTEGERS = ("int64", "int32", "int16", "uint8", "int8")


def _ids(what: str, name: str, ids, x, dims: int):
    import torch

    if str(ids.dtype).replace("torch.", "") not in _INTEGERS or ids.device != x.device:
        raise LossError(f"{what} wants {name} as integers on x's device, not {ids.dtype} on {ids.device}")
    if ids.dim() != x.dim() - 1 + dims or ids.shape[:x.dim() - 1] != x.shape[:-1]:
        raise LossError(f"{what}: {name} {list(ids.shape)} does not go with x {list(x.shape)}")
    return ids.to(torch.int64).contiguous()


def linear_cross_entropy(x, w, target, *, ignore_index: int = -100, reduction: str = "mean"):
    """Softmax cross entropy of the logits ``x @ w.T`` against ``target``, in fp32.

    ``x [..., D]`` and ``w [V, D]`` are both bf16 or both fp16, of any strides (rows that are
    not 16-byte aligned are copied first); ``target [...]`` holds integers.  A token whose
    target is ``ignore_index`` has loss 0 and takes part in no sum, whatever its row of ``x``
    holds; a target outside the vocabulary gives that token a NaN loss (and NaN gradients).
    ``reduction`` is ``mean`` over the tokens that count (0 if none does), ``sum``, or
    ``none`` for a loss per token.  Gradients flow to ``x`` and ``w``, once."""
    x, kept = _check("linear_cross_entropy", x, w, reduction)
    ids = _ids("linear_cross_entropy", "target", target, x, 0)
    kept.k, kept.distill, kept.temperature, kept.ignore = 1, 0, 1.0, int(ignore_index)
    return _autograd().apply(x, w, ids, None, kept)


def linear_distill(x, w, ids, logits, *, temperature: float = 1.0, reduction: str = "mean"):
    """Divergence of the softmax of ``x @ w.T / temperature`` from a teacher's, times
    ``temperature ** 2``, in fp32: per token ``sum_k p_k (log p_k - log q_k)`` over the listed
    entries, with ``p`` the softmax of ``logits / temperature`` over them.

    ``ids [..., K]`` are vocabulary entries and ``logits [..., K]`` the teacher's logits there
    (fp32, bf16 or fp16; no gradient).  An id below 0 is no entry, so lists may differ in
    length; a token without any entry (or with logits of -inf alone) has loss 0 and takes part
    in no sum.  An entry listed twice counts twice.  An id past the vocabulary makes the
    token's loss NaN.  ``x``, ``w`` and ``reduction`` are those of
    :func:`linear_cross_entropy`."""
    import math

    import torch

    what = "linear_distill"
    x, kept = _check(what, x, w, reduction)
    ids = _ids(what, "ids", ids, x, 1)
    if not logits.is_floating_point() or logits.device != x.device or logits.shape != ids.shape:
        raise LossError(f"{what} wants logits as numbers of ids' shape on x's device, not {logits.dtype} "
                        f"{list(logits.shape)} on {logits.device}")
    if logits.requires_grad and torch.is_grad_enabled():
        raise LossError(f"{what} gives the teacher's logits no gradient: detach them")
    if ids.shape[-1] > MAX_TARGETS:
        raise LossError(f"{what}: {ids.shape[-1]} entries a token (at most {MAX_TARGETS})")
    temperature = float(temperature)
    if not (math.isfinite(temperature) and temperature > 0):
        raise LossError(f"{what}: the temperature must be above 0, not {temperature}")
    kept.k, kept.distill, kept.temperature, kept.ignore = ids.shape[-1], 1, temperature, 0
    return _autograd().apply(x, w, ids, logits.detach().float().contiguous(), kept)
