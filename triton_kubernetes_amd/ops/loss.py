"""Python front-end of the output head's losses (``csrc/tk_loss.hip``).

``linear_cross_entropy(x, w, target)`` is the softmax cross entropy of the logits ``x @ w.T``,
and ``linear_distill(x, w, ids, logits)`` their divergence from a teacher's top logits; both
with their gradients (torch autograd).  The ``[tokens, vocabulary]`` logits are not kept: the
forward pass leaves a few numbers a token, and the backward pass computes the logits again, a
piece of the vocabulary at a time.  A caller who has the memory may have them kept in 16 bits
instead (``keep_logits``).  Like ``gemm.gemm_bt`` the losses take torch
tensors on the GPU and queue their work on torch's current stream of that device; nothing
waits for it here, and both directions can be captured into a graph.

A captured backward pass needs everything that it goes through to be made on the capture's
stream.  torch keeps a leaf's gradient node, and its stream, for as long as anything holds that
node: a loss that is alive, a data-parallel reducer, a gradient edge.  Captured then, the pass
would leave that stream behind in the capture, which ends the process.  A call that meets a node
that an earlier call on another stream went through is refused, whatever will be done with its
result: drop what holds the node, or capture with leaves made in the capture
(``x.detach().requires_grad_()``).  A node that only other operations went through before is not
known here, and the same holds for it.
"""

import ctypes
import functools
import struct
from typing import Optional

from .native import NativeUnavailable, load

TILE = 256  # vocabulary entries and tokens of a large tile
SMALL_M, SMALL_N = 128, 64  # of a small one
FEW_ROWS = 512  # tokens whose targets every tile of w's gradient looks for itself
DL_BYTES = 512 << 20  # the backward pass' 16-bit derivative of the logits, per piece
KEEP_BYTES = 4 << 30  # most logits in 16 bits that a call with keep_logits=None keeps for its backward pass
MAX_TARGETS = 1024  # ids of a token's list
MAX_TOKENS = 1 << 20
MAX_WIDTH = 1 << 16
MAX_VOCAB = 1 << 24
MAX_TEMPERATURE_BITS = 32  # the temperature's square, and logits over it, are fp32 numbers
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


class LossError(RuntimeError):
    pass


# struct tkl_args of csrc/tk_loss.hip: n d v k ldx ldw ldg ignore piece fill, dev f16 distill
# reduction, temperature, want small parts, x w ids teacher grad loss kept room codes wc dx
# dw stream
_ARGS = struct.Struct("@10q4if3i13P")

_loaded = None


def _lib():
    global _loaded
    if _loaded is None:
        from .native import require_torch_first

        require_torch_first()
        lib = load("libtk_loss.so")
        lib.tkl_last_error.restype = ctypes.c_char_p
        lib.tkl_kept_bytes.restype = lib.tkl_room_bytes.restype = ctypes.c_longlong
        for call in (lib.tkl_forward, lib.tkl_backward, lib.tkl_kept_bytes, lib.tkl_room_bytes):
            call.argtypes = [ctypes.c_char_p]
        if lib.tkl_args_size() != _ARGS.size:
            raise NativeUnavailable("libtk_loss.so does not match ops/loss.py: run `python -m triton_kubernetes_amd.ops.build`")
        _loaded = lib
    return _loaded


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def pieces(n: int, v: int) -> int:
    """Vocabulary entries of a piece of the backward pass: as many as keep the derivative of
    ``n`` tokens' logits near ``DL_BYTES``, at most half as much again (a second piece for a little
    more costs 2 %: 5000 x 2048 x 60000 in one 4160 us, in two 4228), spread evenly, in whole tiles."""
    count = max(1, min((4 * n * v // DL_BYTES + 1) // 2, -(-v // TILE)))
    # (of a great many tokens a whole tile more can be past that)
    return min(_up(-(-v // count), TILE), max(TILE, 3 * DL_BYTES // (4 * n) // TILE * TILE))


def small_products(n: int, d: int, v: int) -> int:
    """Which products run in small tiles (bits 1: the logits, 2: x's gradient, 4: w's).

    A large tile multiplies faster, a small one wastes less on few tokens and fills more
    compute units.  Measured gain of a small tile over a large one, in us of a whole step at
    bf16 (n x d x v), where the rules turn: logits, 128 x 4096 x 32000 35 of 387, 192 -9, 256 -38;
    4096 x 512 x 1000 21 of 111, 8192 4.  x's gradient, 64 x 4096 x 32000 11, 128 8, 192 -10, 128 x
    4096 x 131072 -50; 2048 x 1024 x 4000 8, 512 x 1024 x 32000 -2, 4096 x 512 x 8000 -3.  w's, 1024 x
    512 x 8000 (64 large tiles) 16, 1024 x 1024 x 6000 (96) 5, 4096 x 1024 x 8000 (128) -7."""

    def tiles(a, b):
        return -(-a // TILE) * -(-b // TILE)

    logits = n <= SMALL_N or tiles(n, v) <= 64 or (tiles(n, v) <= 128 and n <= 2 * SMALL_N)
    dx = n <= SMALL_N or n * d * v <= 3 << 32
    return logits | dx << 1 | (tiles(d, v) <= 96) << 2


def keeps(n: int, d: int, v: int) -> bool:
    """Whether a call with ``keep_logits=None`` keeps the logits, in 16 bits, for its backward pass:
    where that is faster than to compute them again.  A short product is cheaper
    than two passes over its result.  A step at bf16, kept and again, in us: 4096 x 4096 x 32768
    2740 and 3440, 4096 x 512 x 32768 617 and 628, of width 384 558 and 566, 256 515 and 487; few tokens
    read the weight once less (16 x 4096 x 131072 790 and 958, 512 x 256 x 32000 101 and 100)."""
    return (d >= 384 or n <= 512) and 2 * n * v <= KEEP_BYTES


def fill(small: bool) -> int:
    """Most workgroups for x's gradient, among which the vocabulary is split: 3 rounds of a large
    tile for each of the 256 compute units (a step of 5000 x 4000 x 32768, 320 tiles: 4820 us with
    one round, 4370 with 3, 4410 with 5), or one of two small ones."""
    return 512 if small else 768


def weight_parts(n: int, d: int, v: int) -> int:
    """Into how many parts the tokens are split for w's gradient in small tiles: two workgroups for
    each of the 256 compute units, 4 steps of 64 tokens or more each."""
    tiles = -(-d // SMALL_M) * -(-v // SMALL_N)
    return max(1, min(512 // tiles, n // 256, 64))


def kept_bytes(n: int, d: int, lists: int) -> int:
    """Of what the forward pass keeps for the backward pass; ``lists`` entries of a teacher."""
    return 2 * n * _up(d, 64) + 8 + (8 * lists + 36 * n if lists else 24 * n)


def codes_bytes(n: int, v: int, small: bool) -> int:
    """Of the logits kept for the backward pass: 2 bytes each, and a tile's maxima and sums."""
    return 2 * n * _up(v, 256) + part_bytes(n, v, small)


def part_bytes(n: int, v: int, small: bool) -> int:
    return 8 * n * -(-v // (SMALL_M if small else TILE))


def room_bytes(n: int, d: int, piece: int, groups: int, small: int, want: int, lists: int,
               weight: int = 0) -> int:
    """Of the backward pass' workspace: the derivative of a piece's logits (twice with ``small & 8``), fp32 sums of x's
    gradient (as many splits as the tiles of ``groups`` workgroups hold, ``want & 1``), factors,
    the number of splits, residuals and (of more than ``FEW_ROWS`` tokens, ``want & 2``) their lists by
    tile of the vocabulary, fp32 sums of w's gradient (``weight`` rows of them) and x transposed (``want & 2``,
    unless ``small & 4``)."""
    once, halves = n * _up(d, 64), 2 if small & 8 else 1
    tiles = groups * (SMALL_M * SMALL_N if small & 2 else TILE * TILE)
    sums = max(once, min(piece // 512 * once, tiles)) if want & 1 else 0
    rest = 16 * n if lists else 4 * n
    listed = rest + 4 * (piece // TILE + 1) if want & 2 and halves == 1 and n > FEW_ROWS else 0
    return _up(2 * n * piece * halves + 4 * sums + 4 * (n + 2) + rest + listed, 16) \
        + 4 * weight * _up(d, 64) + (2 * _up(d, 64) * _up(n, 64) if want & 2 and not small & 4 else 0)


def _row_strided(w):
    """``w`` with a row stride that the kernels take."""
    if w.shape[0] == 1:
        return w.reshape(-1).contiguous().view(1, -1)  # a lone row's stride may be anything
    return w if w.stride(1) == 1 and w.shape[1] <= w.stride(0) <= 1 << 21 else w.contiguous()


def _room_for_copy(w):
    """Room for a copy of ``w`` with padded rows, where the kernels need one (the forward pass makes
    it, and keeps it for the backward pass)."""
    import torch

    v, d = w.shape
    if d % 8 or w.stride(0) % 8 or w.data_ptr() % 16:
        return torch.empty((v, _up(d, 64)), dtype=w.dtype, device=w.device)
    return None


def _apply(x, w, ids, teacher, plan):
    import torch

    loss = _autograd().apply(x, w, ids, teacher, plan)
    made = loss.grad_fn
    if made is not None:
        stream = torch._C._cuda_getCurrentRawStream(plan.device)
        for node, _ in made.next_functions[:2]:
            # (kept by the node itself, as long as a graph holds it)
            if node is not None and node.metadata.setdefault("tk_loss_stream", stream) != stream:
                with torch.cuda.device(x.device):
                    if torch.cuda.is_current_stream_capturing():
                        del loss, made, node  # or the error's traceback keeps them
                        raise LossError("captured while the gradient node of x or w from an eager graph on another stream "
                                        "lives, through which no gradient can be captured: drop what holds it (an earlier "
                                        "loss, a data-parallel reducer, a gradient edge), or detach x and w in the capture")
    return loss


class _Plan:
    """The sizes and settings of a call, from its forward to its backward pass."""

    __slots__ = ("n", "d", "v", "k", "lead", "distill", "reduction", "temperature", "ignore", "f16", "device", "small", "keep",
                 "kept", "codes", "sums", "piece", "groups", "parts", "room")


_INTEGERS = ("torch.int64", "torch.int32", "torch.int16", "torch.uint8", "torch.int8")


@functools.lru_cache(maxsize=256)
def _plan(what, x, w, ids, logits, reduction, temperature, ignore, keep, grads, rules, precise=False) -> _Plan:
    """The plan of a call whose tensors have these ``(shape, dtype, device)``; calls alike share one
    (``rules``: what else the sizes come from)."""
    (shape, dtype, device), (by, w_type, w_device) = x, w
    if str(dtype) not in ("torch.bfloat16", "torch.float16") or w_type is not dtype:
        raise LossError(f"{what} wants x and w both bf16 or both fp16, not {dtype} and {w_type}")
    if len(shape) < 1 or len(by) != 2 or shape[-1] != by[1]:
        raise LossError(f"{what} wants x [..., D] and w [V, D], not {list(shape)} and {list(by)}")
    if device.type != "cuda" or device != w_device:
        raise LossError(f"{what} wants CUDA tensors on one device, not {device} and {w_device}")
    if reduction not in REDUCTIONS:
        raise LossError(f"unknown reduction '{reduction}' ({' | '.join(REDUCTIONS)})")
    p = _Plan()
    (p.v, p.d), p.lead = by, shape[:-1]
    p.n = n = p.lead.numel()
    d, v = p.d, p.v
    if not (1 <= d <= MAX_WIDTH and 1 <= v <= MAX_VOCAB and n <= MAX_TOKENS):
        raise LossError(f"{what}: {n} tokens of width {d} over {v} entries (at most {MAX_TOKENS}, {MAX_WIDTH}, {MAX_VOCAB})")
    if -(-v // TILE) * -(-n // TILE) >= 1 << 23 or -(-d // 1024) * n >= 1 << 24:
        raise LossError(f"{what}: {n} tokens of width {d} over {v} entries: tokens x vocabulary must be below 2^39, "
                        "tokens x width below 2^34")
    id_shape, id_type, id_device = ids
    name = "target" if logits is None else "ids"
    if str(id_type) not in _INTEGERS or id_device != device:
        raise LossError(f"{what} wants {name} as integers on x's device, not {id_type} on {id_device}")
    if (id_shape if logits is None else id_shape[:-1]) != p.lead or (logits is not None and len(id_shape) == 0):
        raise LossError(f"{what}: {name} {list(id_shape)} does not go with x {list(shape)}")
    p.k, p.distill = 1, 0
    if logits is not None:
        if not logits[1].is_floating_point or logits[2] != device or logits[0] != id_shape:
            raise LossError(f"{what} wants logits as numbers of ids' shape on x's device, not {logits[1]} {list(logits[0])} "
                            f"on {logits[2]}")
        p.k, p.distill = id_shape[-1], 1
        if p.k > MAX_TARGETS:
            raise LossError(f"{what}: {p.k} entries a token (at most {MAX_TARGETS})")
        if not 2.0 ** -MAX_TEMPERATURE_BITS <= temperature <= 2.0 ** MAX_TEMPERATURE_BITS:  # (not if it is NaN)
            raise LossError(f"{what}: the temperature must be 2^-{MAX_TEMPERATURE_BITS} to 2^{MAX_TEMPERATURE_BITS}, "
                            f"not {temperature}")
    if not -(1 << 63) <= ignore < 1 << 63:
        raise LossError(f"{what}: no target can be {ignore}")
    p.reduction, p.temperature, p.ignore = REDUCTIONS[reduction], temperature, ignore
    if precise and keep:
        raise LossError(f"{what}: kept logits are rounded, so a precise gradient has to compute them again")
    p.f16, p.device = str(dtype) == "torch.float16", device.index
    if n and p.k:
        p.small = small_products(n, d, v) | (8 if precise else 0)
        p.keep = grads and not precise and (keeps(n, d, v) if keep is None else bool(keep))
        p.kept = _up(kept_bytes(n, d, n * p.k if p.distill else 0), 256)
        p.codes = p.kept if p.keep else 0  # the logits lie behind the rest
        p.sums = part_bytes(n, v, bool(p.small & 1))
        if p.keep:
            p.kept += codes_bytes(n, v, bool(p.small & 1))
        p.piece = pieces(n, v)
        if precise:  # half of the piece's memory for each part
            p.piece = min(p.piece, pieces(2 * n, v))
        p.groups = fill(bool(p.small & 2))
        parts = weight_parts(n, d, v) if p.small & 4 and p.piece >= v else 1
        p.parts = (1, 1, parts, parts)  # by the gradients that are wanted
        p.room = tuple(room_bytes(n, d, p.piece, p.groups, p.small, want, p.distill,
                                  p.parts[want] * v if p.parts[want] > 1 else 0) for want in range(4))
    return p


def _planned(what, x, w, ids, logits, reduction, temperature, ignore, keep, precise):
    import torch

    grads = torch.is_grad_enabled() and (x.requires_grad or w.requires_grad)
    rules = (small_products, keeps, pieces, fill, weight_parts, DL_BYTES, KEEP_BYTES)
    return _plan(what, (x.shape, x.dtype, x.device), (w.shape, w.dtype, w.device), (ids.shape, ids.dtype, ids.device),
                 None if logits is None else (logits.shape, logits.dtype, logits.device), reduction, temperature, ignore,
                 keep, grads, rules, bool(precise))


def _ids(ids):
    import torch

    return ids if ids.dtype is torch.int64 and ids.is_contiguous() else ids.to(torch.int64).contiguous()


_function = None


def _autograd():
    """The autograd function (torch is imported on first use)."""
    global _function
    if _function is not None:
        return _function
    import torch

    lib, stream_of = _lib(), torch._C._cuda_getCurrentRawStream

    def gradients(ctx, grad):
        plan = ctx.plan
        need = ctx.needs_input_grad
        want = (1 if need[0] else 0) | (2 if need[1] else 0)
        n, d, v, k = plan.n, plan.d, plan.v, plan.k
        if n == 0 or k == 0:
            x, w = ctx.saved_tensors
            return (torch.zeros_like(x) if want & 1 else None, torch.zeros_like(w) if want & 2 else None, None, None,
                    None)
        w, kept, copy, ids = ctx.saved_tensors
        if not plan.reduction:
            grad = grad.reshape(-1)
        if grad.dtype is not torch.float32:
            grad = grad.float()
        plain = _row_strided(w) if copy is None else copy
        room = kept.new_empty(plan.room[want])
        dx = w.new_empty((n, d)) if want & 1 else None
        dw = w.new_empty((v, d)) if want & 2 else None
        at = kept.data_ptr()
        args = _ARGS.pack(n, d, v, k, 0, plain.stride(0), 0 if plan.reduction else grad.stride(0), plan.ignore,
                          plan.piece, plan.groups, plan.device, plan.f16, plan.distill, plan.reduction, plan.temperature,
                          want, plan.small, plan.parts[want], 0, plain.data_ptr(), 0 if ids is None else ids.data_ptr(), 0,
                          grad.data_ptr(), 0, at, room.data_ptr(), at + plan.codes if plan.codes else 0,
                          0 if copy is None else copy.data_ptr(), 0 if dx is None else dx.data_ptr(),
                          0 if dw is None else dw.data_ptr(), stream_of(plan.device))
        if want and lib.tkl_backward(args) != 0:
            raise LossError(lib.tkl_last_error().decode())
        if dx is not None and len(plan.lead) != 1:
            dx = dx.view(*plan.lead, d)
        return dx, dw, None, None, None

    class Once(torch.autograd.Function):
        """A gradient that was made with create_graph: to differentiate it again is an error."""

        @staticmethod
        def forward(ctx, g, w):
            return g.view_as(g)

        @staticmethod
        def backward(ctx, grad):
            raise LossError("the head's losses have no second derivative")

    class HeadLoss(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, ids, teacher, plan):
            n, d, v, k = plan.n, plan.d, plan.v, plan.k
            ctx.plan = plan
            loss = x.new_empty(() if plan.reduction else plan.lead, dtype=torch.float32)
            if n == 0 or k == 0:  # nothing has a loss
                ctx.save_for_backward(x, w)
                return loss.zero_()
            if len(plan.lead) != 1:
                x = x.reshape(n, d)
            ldx, step = x.stride()
            if step != 1:
                x = x.contiguous()
                ldx = x.stride(0)
            plain = _row_strided(w)
            copy = _room_for_copy(plain)
            kept = x.new_empty(plan.kept, dtype=torch.uint8)
            at = kept.data_ptr()
            if plan.keep:
                sums, codes = None, at + plan.codes
            else:
                sums, codes = x.new_empty(plan.sums, dtype=torch.uint8), 0
            args = _ARGS.pack(n, d, v, k, ldx, plain.stride(0), 0, plan.ignore, 0, 0, plan.device, plan.f16, plan.distill,
                              plan.reduction, plan.temperature, 0, plan.small, 1, x.data_ptr(), plain.data_ptr(),
                              ids.data_ptr(), 0 if teacher is None else teacher.data_ptr(), 0, loss.data_ptr(), at,
                              codes or sums.data_ptr(), codes, 0 if copy is None else copy.data_ptr(), 0, 0,
                              stream_of(plan.device))
            if lib.tkl_forward(args) != 0:
                raise LossError(lib.tkl_last_error().decode())
            ctx.save_for_backward(w, kept, copy, ids if plan.distill else None)  # (kept has the targets)
            return loss

        @staticmethod
        def backward(ctx, grad):
            if not torch.is_grad_enabled():
                return gradients(ctx, grad)
            with torch.no_grad():
                grads = gradients(ctx, grad)
            return tuple(None if g is None else Once.apply(g.requires_grad_(), ctx.saved_tensors[0]) for g in grads)

    _function = HeadLoss
    return _function


def linear_cross_entropy(x, w, target, *, ignore_index: int = -100, reduction: str = "mean",
                         keep_logits: Optional[bool] = False, precise_grad: bool = False):
    """Softmax cross entropy of the logits ``x @ w.T`` against ``target``, in fp32.

    ``x [..., D]`` and ``w [V, D]`` are both bf16 or both fp16, of any strides (rows that are
    not 16-byte aligned are copied first); ``target [...]`` holds integers.  A token whose
    target is ``ignore_index`` has loss 0 and takes part in no sum, whatever its row of ``x``
    holds; a target outside the vocabulary gives that token a NaN loss (and NaN gradients).
    ``reduction`` is ``mean`` over the tokens that count (0 if none does), ``sum``, or
    ``none`` for a loss per token.  Gradients flow to ``x`` and ``w``, once.

    Between the passes the logits are not kept.  ``keep_logits=True`` keeps them, 2 bytes each
    for as long as the loss lives, instead of computing them again, and ``None`` does so up to
    ``KEEP_BYTES`` where :func:`keeps` finds that faster.  Kept logits are rounded: a probability
    is then off by up to 8.5e-5 of itself, 3.4e-4 below 2^-8 of its tile's largest and 2.7e-3
    below 2^-24, which joins the rounding of the gradient's operands.

    These are in 16 bits: ``x``, ``w``, and the derivative of the logits, rounded to their type, of
    which the targets get back what that took.  The gradients are off by 1.00 times what rounding
    them once costs where the targets are most of the derivative, as in training; up to 1.35 times was
    seen where a teacher's lists spread it.  ``precise_grad=True`` multiplies the derivative in two
    16-bit parts instead, so that little but the result's own rounding is left (1.00 times in any
    case), for about half as much time again."""
    plan = _planned("linear_cross_entropy", x, w, target, None, reduction, 1.0, int(ignore_index), keep_logits,
                    precise_grad)
    return _apply(x, w, _ids(target), None, plan)


def linear_distill(x, w, ids, logits, *, temperature: float = 1.0, reduction: str = "mean",
                   keep_logits: Optional[bool] = False, precise_grad: bool = False):
    """Divergence of the softmax of ``x @ w.T / temperature`` from a teacher's, times
    ``temperature ** 2``, in fp32: per token ``sum_k p_k (log p_k - log q_k)`` over the listed
    entries, with ``p`` the softmax of ``logits / temperature`` over them.

    ``ids [..., K]`` are vocabulary entries and ``logits [..., K]`` the teacher's logits there
    (fp32, bf16 or fp16; no gradient).  An id below 0 is no entry, so lists may differ in
    length; a token without any entry (or with logits of -inf alone) has loss 0 and takes part
    in no sum.  An entry listed twice counts twice.  An id past the vocabulary makes the
    token's loss NaN.  The temperature is 2^-32 to 2^32; the loss has the rounding of fp32
    logarithms times its square.  ``x``, ``w``, ``reduction``, ``keep_logits`` and ``precise_grad`` are
    those of :func:`linear_cross_entropy`."""
    import torch

    plan = _planned("linear_distill", x, w, ids, logits, reduction, float(temperature), 0, keep_logits,
                    precise_grad)
    if logits.requires_grad and torch.is_grad_enabled():
        raise LossError("linear_distill gives the teacher's logits no gradient: detach them")
    if torch.autograd.forward_ad._current_level >= 0 and torch.autograd.forward_ad.unpack_dual(logits).tangent is not None:
        raise LossError("linear_distill gives the teacher's logits no gradient: detach them")
    return _apply(x, w, _ids(ids), logits.detach().float().contiguous(), plan)
