"""Losses over a vocabulary, on the ``det_vocab.hip`` kernels.

    linear_cross_entropy(x, W, target[, b])            CE(x W^T + b, target)
    linear_topk_distill(x, W, teacher, index[, b])     T^2 KL(teacher's top logits || softmax((x W^T + b) / T))
    topk_distill(logits, teacher, index)               the same for logits that are there already

The ``linear_`` forms are a language model's output layer and its loss in one, walking the vocabulary in
chunks: the [rows, V] logits are never in memory.  The forward reduces each tile of them to a maximum and
a sum of exponentials; the backward turns a chunk at a time into the logits' gradient and multiplies that
into the gradients of ``x`` and ``W``.  It makes a chunk from exponentials that the forward held, of as many
chunks as ``hold_bytes`` has room for, and from the logits computed again past those.  Rows that are
ignored cost nothing.  Losses are fp32; sums, softmax statistics and gradients are accumulated in fp32; a
chunk's logit gradient is held in the operands' type (fp32: two fp16 planes, 22 bits), exponentials in 16
bits with a step of 2^-11 down to 2^-31 of a tile's largest (for fp32 operands and with label smoothing: in
fp32; with ``hold_bytes=0`` none are).

GPU tensors (bf16, fp16, fp32) always run on the kernels; what those do not cover is refused.  CPU
tensors run the plain composite below.  The kernels are differentiable once.

fp32 operands are multiplied as two fp16 planes each, under a power of two: a row's own for ``x`` in the logits,
one for all words of ``W`` (those that a bias of -inf takes out do not count), one for all kept rows of ``x``
in ``W``'s gradient.  Entries more than 2^16 below the largest under the same scale are held to 2^-39 of that
one instead of 2^-23 of themselves.

Memory of a ``linear_`` call: between forward and backward at most ``hold_bytes`` (2 or, where they are fp32, 4
bytes a logit) and two percent more, the kept rows of ``x`` once more, 8 K bytes a row, and weights that had to be packed
(fp32, or rows that 16 bytes do not divide) up to 4 GiB of them; in the backward 512 MiB for a chunk's logit
gradient, fp32 sums of ``x``'s gradient, and for fp32, and fp16 with ``reduction="none"``, the kept rows of ``x``
again.  Under ``torch.no_grad()`` none of these exponentials.
"""
import ctypes
import math
from typing import Any, Optional

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from determined_1_amd.ops import _lib
from determined_1_amd.ops.arena import landing_buffer
from determined_1_amd.ops.functional import dtype_code
from determined_1_amd.ops.transformer import _autocast, _null, _ptr, _stream

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
HOLD_BYTES = 2 << 30  # under one percent of the card's memory
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class _HeadParams(ctypes.Structure):
    """Mirror of ``DetVocabHead`` (det_vocab.hip)."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "w", "bias", "target", "index", "teacher", "dx", "dw", "db", "gout",
                                                "loss", "kept", "ws")]
                + [(n, ctypes.c_int64) for n in ("ws_bytes", "kept_bytes", "x_ld", "w_ld", "index_ld", "teacher_ld", "ignore",
                                                "hold_bytes")]
                + [(n, ctypes.c_int32) for n in ("N", "D", "V", "K", "dtype", "bias_dt", "wide", "teacher_dt", "reduction")]
                + [("inv_t", ctypes.c_float), ("smooth", ctypes.c_float)])


class _LogitParams(ctypes.Structure):
    """Mirror of ``DetVocabLogits`` (det_vocab.hip)."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("z", "index", "teacher", "dz", "gout", "loss", "kept")]
                + [(n, ctypes.c_int64) for n in ("kept_bytes", "z_ld", "index_ld", "teacher_ld", "dz_ld")]
                + [(n, ctypes.c_int32) for n in ("N", "V", "K", "dtype", "wide", "teacher_dt", "reduction")]
                + [("inv_t", ctypes.c_float)])


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """[..., C] as [rows, C] with a unit last stride (a view where the layout allows it)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 else t.contiguous()


def _apart(teacher: torch.Tensor) -> torch.Tensor:
    return teacher.detach() if teacher.requires_grad else teacher


def _buffer(nbytes: int, like: torch.Tensor, what: str) -> torch.Tensor:
    if nbytes < 0:
        raise ValueError(f"{what}: sizes out of the kernels' range")
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device)


def _on(t: torch.Tensor):
    """The tensor's device as the current one (a kernel is launched on the current device)."""
    return _null() if t.device.index == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def _traced(*ts: Optional[torch.Tensor]) -> bool:
    """Whether autograd has to see the call (forward mode: to refuse it)."""
    return forward_ad._current_level >= 0 or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts))


def _once(fn):
    """``once_differentiable`` without its cost (5 us a call) where no second derivative can be asked for."""
    guarded = torch.autograd.function.once_differentiable(fn)
    return staticmethod(lambda ctx, gout: (guarded if torch.is_grad_enabled() else fn)(ctx, gout))


class _Head(torch.autograd.Function):
    """x [N, D], weight [V, D]: unit last strides; target [N], or index and teacher [N, K]."""

    @staticmethod
    def run(x, weight, bias, target, teacher, index, opts):
        """(loss, what the backward pass needs, the call)"""
        ignore, smooth, heat, reduction, hold_bytes = opts
        p = _HeadParams()
        p.N, p.D = x.shape
        p.V = weight.shape[0]
        p.x, p.w, p.x_ld, p.w_ld = x.data_ptr(), weight.data_ptr(), x.stride(0), weight.stride(0)
        p.dtype = dtype_code(x.dtype)
        if bias is not None:
            p.bias, p.bias_dt = bias.data_ptr(), dtype_code(bias.dtype)
        p.ignore, p.smooth, p.inv_t, p.reduction, p.hold_bytes = ignore, smooth, 1.0 / heat, _REDUCTIONS[reduction], hold_bytes
        if target is not None:
            p.target, p.K, p.wide = target.data_ptr(), 1, target.dtype == torch.int64
        else:
            p.index, p.teacher, p.K = index.data_ptr(), teacher.data_ptr(), index.shape[1]
            p.index_ld, p.teacher_ld = index.stride(0), teacher.stride(0)
            p.wide, p.teacher_dt = index.dtype == torch.int64, dtype_code(teacher.dtype)
        ref, lib = ctypes.byref(p), _lib.get_lib()
        loss = torch.empty(p.N if reduction == "none" else (), dtype=torch.float32, device=x.device)
        kept = _buffer(lib.det_vocab_head_bytes(ref, 0), x, "vocab_loss")
        ws = _buffer(lib.det_vocab_head_bytes(ref, 1), x, "vocab_loss")
        p.loss, p.kept, p.ws = loss.data_ptr(), kept.data_ptr(), ws.data_ptr()
        p.kept_bytes, p.ws_bytes = kept.numel(), ws.numel()
        with _on(x):
            _lib.check(lib.det_vocab_head_forward(_stream(x), ref), "det_vocab_head_forward")
        return loss, kept, p

    @staticmethod
    def forward(ctx, x, weight, bias, target, teacher, index, opts):  # type: ignore[override]
        loss, kept, ctx.params = _Head.run(x, weight, bias, target, teacher, index, opts)
        ctx.save_for_backward(x, weight, bias, target, teacher, index, kept)
        return loss

    @_once
    def backward(ctx, gout):  # type: ignore[override]
        x, weight, bias, target, teacher, index, kept = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        p = _HeadParams.from_buffer_copy(ctx.params)
        # the pointers anew: saved-tensor hooks may have moved what was saved
        p.x, p.w, p.x_ld, p.w_ld, p.kept = x.data_ptr(), weight.data_ptr(), x.stride(0), weight.stride(0), kept.data_ptr()
        p.bias, p.target = _ptr(bias), _ptr(target)
        if index is not None:
            p.index, p.teacher, p.index_ld, p.teacher_ld = index.data_ptr(), teacher.data_ptr(), index.stride(0), teacher.stride(0)
        gout = gout.float().contiguous()
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
        dw = db = None
        if need_w:
            dw = landing_buffer(weight)
            if dw is None or dw.dtype != weight.dtype or not dw.is_contiguous() or dw.shape != weight.shape:
                dw = torch.empty_like(weight, memory_format=torch.contiguous_format)
        if need_b:
            db = torch.empty_like(bias)
        p.dx, p.dw, p.db, p.gout = _ptr(dx), _ptr(dw), _ptr(db), gout.data_ptr()
        ref, lib = ctypes.byref(p), _lib.get_lib()
        ws = _buffer(lib.det_vocab_head_bytes(ref, 2), x, "vocab_loss")
        p.ws, p.ws_bytes = ws.data_ptr(), ws.numel()
        with _on(x):
            _lib.check(lib.det_vocab_head_backward(_stream(x), ref), "det_vocab_head_backward")
        return dx, dw, db, None, None, None, None


class _Logits(torch.autograd.Function):
    """logits [N, V], teacher and index [N, K]: unit last strides."""

    @staticmethod
    def run(z, teacher, index, heat, reduction):
        """(loss, what the backward pass needs, the call)"""
        p = _LogitParams()
        p.N, p.V = z.shape
        p.z, p.index, p.teacher, p.K = z.data_ptr(), index.data_ptr(), teacher.data_ptr(), index.shape[1]
        p.z_ld, p.index_ld, p.teacher_ld = z.stride(0), index.stride(0), teacher.stride(0)
        p.dtype, p.wide, p.teacher_dt = dtype_code(z.dtype), index.dtype == torch.int64, dtype_code(teacher.dtype)
        p.reduction, p.inv_t = _REDUCTIONS[reduction], 1.0 / heat
        ref, lib = ctypes.byref(p), _lib.get_lib()
        loss = torch.empty(p.N if reduction == "none" else (), dtype=torch.float32, device=z.device)
        kept = _buffer(lib.det_vocab_logits_bytes(ref), z, "topk_distill")
        p.loss, p.kept, p.kept_bytes = loss.data_ptr(), kept.data_ptr(), kept.numel()
        with _on(z):
            _lib.check(lib.det_vocab_logits_forward(_stream(z), ref), "det_vocab_logits_forward")
        return loss, kept, p

    @staticmethod
    def forward(ctx, z, teacher, index, heat, reduction):  # type: ignore[override]
        loss, kept, ctx.params = _Logits.run(z, teacher, index, heat, reduction)
        ctx.save_for_backward(z, teacher, index, kept)
        return loss

    @_once
    def backward(ctx, gout):  # type: ignore[override]
        z, teacher, index, kept = ctx.saved_tensors
        p = _LogitParams.from_buffer_copy(ctx.params)
        # the pointers anew: saved-tensor hooks may have moved what was saved
        p.z, p.index, p.teacher, p.kept = z.data_ptr(), index.data_ptr(), teacher.data_ptr(), kept.data_ptr()
        p.z_ld, p.index_ld, p.teacher_ld = z.stride(0), index.stride(0), teacher.stride(0)
        gout = gout.float().contiguous()
        dz = torch.empty_like(z, memory_format=torch.contiguous_format)
        p.gout, p.dz, p.dz_ld = gout.data_ptr(), dz.data_ptr(), dz.stride(0)
        with _on(z):
            _lib.check(_lib.get_lib().det_vocab_logits_backward(_stream(z), ctypes.byref(p)), "det_vocab_logits_backward")
        return dz, None, None, None, None


# ------------------------------------------------------------------------------------------------
# plain composite (CPU tensors)
# ------------------------------------------------------------------------------------------------
def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


def _reduce(rows: torch.Tensor, kept: torch.Tensor, reduction: str) -> torch.Tensor:
    rows = torch.where(kept, rows, torch.zeros_like(rows))
    if reduction == "none":
        return rows
    return rows.sum() / kept.sum().clamp(min=1) if reduction == "mean" else rows.sum()


def _pick(logp: torch.Tensor, index: torch.Tensor, there: torch.Tensor) -> torch.Tensor:
    """logp at each index; NaN for one outside the vocabulary, 0 where there is no entry."""
    v = logp.shape[-1]
    got = logp.gather(1, index.long().clamp(0, v - 1))
    outside = torch.zeros_like(got).masked_fill_(there & ((index < 0) | (index >= v)), math.nan)
    got = got * (1.0 + outside)  # the gradient is NaN too
    return torch.where(there, got, torch.zeros_like(got))


def _there(teacher: torch.Tensor, index: torch.Tensor) -> torch.Tensor:
    return (index >= 0) & (teacher != -math.inf)


def _plain_ce(z: torch.Tensor, target: torch.Tensor, ignore: int, smooth: float, reduction: str) -> torch.Tensor:
    kept = target != ignore
    z = torch.where(kept[:, None], z, torch.zeros_like(z))
    logp = F.log_softmax(z, dim=1)
    picked = _pick(logp, target[:, None], kept[:, None])[:, 0]
    if smooth == 1.0:  # the target does not count, not even one of logit -inf
        picked = torch.where(picked.isnan(), picked, torch.zeros_like(picked))
    rows = -(1.0 - smooth) * picked
    if smooth:
        rows = rows - smooth * logp.mean(dim=1)
    return _reduce(rows, kept, reduction)


def _plain_distill(z: torch.Tensor, teacher: torch.Tensor, index: torch.Tensor, heat: float, reduction: str) -> torch.Tensor:
    t = _wide(teacher).to(z.dtype) / heat
    there = _there(t, index)
    kept = there.any(dim=1)
    z = torch.where(kept[:, None], z, torch.zeros_like(z))
    logp = F.log_softmax(z / heat, dim=1)
    logq = F.log_softmax(torch.where(there, t, torch.full_like(t, -math.inf)).masked_fill(~kept[:, None], 0.0), dim=1)
    q = torch.where(there, logq.exp(), torch.zeros_like(logq))
    there = there & (q != 0)
    rows = torch.where(there, q * (logq.masked_fill(~there, 0.0) - _pick(logp, index, there)), torch.zeros_like(q)).sum(dim=1)
    bad = torch.zeros_like(rows).masked_fill_((index >= z.shape[1]).any(dim=1), math.nan)
    rows = rows * (1.0 + bad)
    return _reduce(rows * heat * heat, kept, reduction)


# ------------------------------------------------------------------------------------------------
# public API
# ------------------------------------------------------------------------------------------------
def _refuse(what: str, message: str, error: Any = ValueError) -> None:
    raise error(f"{what}: {message}")


def _check_common(what: str, reduction: str, first: torch.Tensor, *ts: Optional[torch.Tensor]) -> None:
    if reduction not in _REDUCTIONS:
        _refuse(what, f"reduction {reduction!r} is none of {sorted(_REDUCTIONS)}")
    device = first.device
    for t in ts:
        if t is not None and t.device != device:
            _refuse(what, f"tensors on {device} and {t.device}")
    if device.type not in ("cpu", "cuda"):
        _refuse(what, f"no kernels for {device}")


def _check_float(what: str, x: torch.Tensor, name: str) -> None:
    if x.dtype not in _FLOATS and not (x.dtype == torch.float64 and x.device.type == "cpu"):
        _refuse(what, f"{name} is {x.dtype}: bfloat16, float16 or float32 expected", TypeError)


def _check_head(what: str, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> None:
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        _refuse(what, f"x [..., D] and weight [V, D] expected, got {tuple(x.shape)} and {tuple(weight.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        _refuse(what, f"bias of {weight.shape[0]} words expected, got {tuple(bias.shape)}")
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        return  # which casts them alike
    _check_float(what, x, "x")
    if weight.dtype != x.dtype:
        _refuse(what, f"x is {x.dtype} and weight {weight.dtype}", TypeError)
    if bias is not None and bias.dtype not in (x.dtype, torch.float32):
        _refuse(what, f"x is {x.dtype} and bias {bias.dtype}", TypeError)


def _check_lists(what: str, lead: torch.Size, teacher: torch.Tensor, index: torch.Tensor, heat: float) -> None:
    if index.shape[:-1] != lead or index.dim() == 0 or index.shape[-1] == 0 or teacher.shape != index.shape:
        _refuse(what, f"teacher_logits and teacher_index {tuple(lead) + ('K',)} expected, got {tuple(teacher.shape)} and "
                      f"{tuple(index.shape)}")
    if index.dtype not in (torch.int32, torch.int64):
        _refuse(what, f"teacher_index is {index.dtype}: int32 or int64 expected", TypeError)
    _check_float(what, teacher, "teacher_logits")
    if not 2.0 ** -20 <= heat <= 2.0 ** 20:
        _refuse(what, f"temperature {heat} is not within [2^-20, 2^20]")


def _bytes(what: str, hold_bytes: int) -> int:
    if not isinstance(hold_bytes, int) or not 0 <= hold_bytes < 2 ** 63:
        _refuse(what, f"hold_bytes {hold_bytes!r} is not a number of bytes")
    return hold_bytes


def _empty(reduction: str, lead: torch.Size, *ts: Optional[torch.Tensor]) -> torch.Tensor:
    """The loss of no rows: 0, with gradients of zeros, whatever the tensors hold."""
    zero = sum(_wide(t.narrow(0, 0, 0)).sum() for t in ts if t is not None)
    return zero if reduction != "none" else zero.expand(lead)


def _linear(x, weight, bias, target, teacher, index, opts, lead) -> torch.Tensor:
    ac = x.is_cuda and torch.is_autocast_enabled("cuda")
    if ac:
        (x, weight, bias), _ = _autocast(x, weight, bias)
    if x.numel() == 0:
        return _empty(opts[3], lead, x, weight, bias)
    x2 = _rows_of(x)
    if target is not None:
        target = target.reshape(-1).contiguous() if target.dim() != 1 or not target.is_contiguous() else target
    else:
        teacher, index = _rows_of(_apart(teacher)), _rows_of(index)
    if x.device.type == "cpu":
        kept = target != opts[0] if target is not None else _there(teacher, index).any(dim=1)
        wide = _wide(x2).masked_fill(~kept[:, None], 0.0)  # what an ignored row holds does not matter
        z = F.linear(wide, _wide(weight), None if bias is None else _wide(bias).to(wide.dtype))
        loss = (_plain_ce(z, target, opts[0], opts[1], opts[3]) if target is not None
                else _plain_distill(z, teacher, index, opts[2], opts[3]))
    else:
        if weight.stride(1) != 1:
            weight = weight.contiguous()
        if bias is not None and bias.stride(0) != 1:
            bias = bias.contiguous()
        if not _traced(x2, weight, bias):
            loss = _Head.run(x2, weight, bias, target, teacher, index, (*opts[:4], 0))[0]  # nothing to hold anything for
        else:
            with torch.autocast("cuda", enabled=False) if ac else _null():
                loss = _Head.apply(x2, weight, bias, target, teacher, index, opts)
    return loss if opts[3] != "none" or len(lead) == 1 else loss.reshape(lead)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                         ignore_index: int = -100, label_smoothing: float = 0.0, reduction: str = "mean",
                         hold_bytes: int = HOLD_BYTES) -> torch.Tensor:
    """``F.cross_entropy(F.linear(x, weight, bias), target, ...)`` without the logits.

    x [..., D], weight [V, D], bias [V] (x's type or fp32), target [...] int32 or int64.  Rows whose target is
    ``ignore_index`` have loss 0, no gradient, and take no work; a mean over none of them is 0.  A target
    outside the vocabulary gives its row (and a mean or sum) a NaN loss and NaN gradients: nothing is read
    out of bounds, and no host check waits for the GPU.  With ``reduction="none"`` each row's gradient by x has
    the precision of its own incoming derivative, however small beside the others, and one that is not finite
    spoils its own row (and the gradients that sum over rows).  With ``reduction="none"`` under ``torch.no_grad()``
    it scores tokens: the loss [...] is each target's negative log-probability.  ``hold_bytes`` bounds what a
    call holds of its logits' exponentials for its backward pass; 0 recomputes all of them there."""
    what = "linear_cross_entropy"
    _check_common(what, reduction, x, weight, target, bias)
    _check_head(what, x, weight, bias)
    lead = x.shape[:-1]
    if target.shape != lead:
        _refuse(what, f"target {tuple(lead)} expected, got {tuple(target.shape)}")
    if target.dtype not in (torch.int32, torch.int64):
        _refuse(what, f"target is {target.dtype}: int32 or int64 expected", TypeError)
    if not 0.0 <= label_smoothing <= 1.0:
        _refuse(what, f"label_smoothing {label_smoothing} is not within [0, 1]")
    ignore = int(ignore_index)
    if not -2 ** 63 <= ignore < 2 ** 63:
        _refuse(what, f"ignore_index {ignore_index} is not of 64 bits")
    opts = (ignore, float(label_smoothing), 1.0, reduction, _bytes(what, hold_bytes))
    return _linear(x, weight, bias, target, None, None, opts, lead)


def linear_topk_distill(x: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor,
                        bias: Optional[torch.Tensor] = None, *, temperature: float = 1.0, reduction: str = "mean",
                        hold_bytes: int = HOLD_BYTES) -> torch.Tensor:
    """``topk_distill(F.linear(x, weight, bias), teacher_logits, teacher_index, ...)`` without the logits.

    x [..., D], weight [V, D], bias [V]; the lists [..., K] as in ``topk_distill``, of up to a few hundred words (a
    step of 2,048 rows of 2,048 against 32,000 words: 0.95 ms for K = 64, 1.2 for 256, 3.2 for 1,024, 23 for
    4,096); ``hold_bytes`` and rows with ``reduction="none"`` as in ``linear_cross_entropy``."""
    what = "linear_topk_distill"
    _check_common(what, reduction, x, weight, teacher_logits, teacher_index, bias)
    _check_head(what, x, weight, bias)
    lead, heat = x.shape[:-1], float(temperature)
    _check_lists(what, lead, teacher_logits, teacher_index, heat)
    opts = (-100, 0.0, heat, reduction, _bytes(what, hold_bytes))
    return _linear(x, weight, bias, None, teacher_logits, teacher_index, opts, lead)


def topk_distill(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor, *, temperature: float = 1.0,
                 reduction: str = "mean") -> torch.Tensor:
    """Distillation from a teacher's top logits: ``T^2 sum_k q_k (log q_k - log p[index_k])`` a row, with
    ``p = softmax(logits / T)`` over the vocabulary and ``q = softmax(teacher_logits / T)`` over the list.

    logits [..., V]; teacher_logits and teacher_index [..., K] (int32 or int64; ``torch.topk``'s values and
    indices), no gradient for them.  Entries with a negative index or a logit of -inf are absent, so lists
    may be of any length up to K; a row without an entry has loss 0 and no gradient and does not count in a
    mean; a mean over none is 0.  A word that is listed twice has the sum of its shares.  An index past the
    vocabulary gives its row a NaN loss and NaN gradients.  Meant for lists of up to a few hundred words: the
    gradient's work on a list grows with K^2 (2,048 rows of 32,000 bf16 logits: 0.1 ms for K up to 256, 0.4 ms for
    1,024, 5 ms for 4,096)."""
    what = "topk_distill"
    _check_common(what, reduction, logits, teacher_logits, teacher_index)
    if logits.dim() < 1 or logits.shape[-1] == 0:
        _refuse(what, f"logits [..., V] expected, got {tuple(logits.shape)}")
    _check_float(what, logits, "logits")
    lead, heat = logits.shape[:-1], float(temperature)
    _check_lists(what, lead, teacher_logits, teacher_index, heat)
    if logits.numel() == 0:
        return _empty(reduction, lead, logits)
    z, teacher, index = _rows_of(logits), _rows_of(_apart(teacher_logits)), _rows_of(teacher_index)
    if logits.device.type == "cpu":
        loss = _plain_distill(_wide(z), teacher, index, heat, reduction)
    else:
        loss = _Logits.apply(z, teacher, index, heat, reduction) if _traced(z) else _Logits.run(z, teacher, index, heat, reduction)[0]
    return loss if reduction != "none" or len(lead) == 1 else loss.reshape(lead)
