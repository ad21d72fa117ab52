"""Losses of post-training on vocabulary-parallel logits: a preference loss over pairs of sequences and a clipped policy loss
with a KL term.

Both are functions of the log-probabilities that a policy gives the labels of the positions whose ``loss_mask`` is not zero.
Positions of mask zero -- prompts, padding -- are not read: their logits may hold anything and their gradient is zero.  On a GPU
the logits are streamed once for the loss and once for its gradient (``csrc/policy_losses.cu``), in their own type and memory
order; the sums over a sequence and everything behind them are in 64 bits.  ``*_ref`` are the same losses in plain PyTorch: the
CPU path and the statement the kernels are tested against.

Reference counterparts: the DPO and REINFORCE objectives of ``megatron/training.py:533-939``, which form ``[b, s, V]``
log-probabilities in fp32.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F

from . import native
from .functional import _DT, _k, device_of, once

KL_KINDS = {"kl": 1, "abs": 2, "mse": 3, "k3": 4, "full": 5}

_P, _I, _L, _D, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_double, ctypes.c_float
native._ARGTYPES.update({
    "neox_vocab_splits": [_L, _I, _I, _I],
    "neox_loss_pieces": [_I],
    "neox_vocab_stats": [_P, _L, _L, _P, _L, _L, _P, _P, _I, _I, _I, _L, _I, _I, _P, _P, _P, _P, _P],
    "neox_preference_loss": [_P, _P, _I, _I, _P, _P, _P, _I, _I, _I, _L, _D, _D, _P, _P, _P, _P, _P, _P, _P, _P],
    "neox_policy_loss": [_P, _P, _P, _I, _I, _P, _P, _P, _L, _L, _P, _P, _I, _I, _I, _L, _I, _I, _D, _D, _D, _P, _P, _P, _P, _P, _P, _P,
                         _P, _P],
    "neox_vocab_grad": [_P, _L, _L, _P, _L, _L, _P, _L, _L, _P, _P, _P, _P, _P, _P, _P, _P, _F, _I, _I, _I, _L, _I, _P],
})
native._CountingLib._NOT_LAUNCHES.update({"neox_vocab_splits", "neox_loss_pieces"})


class PreferenceLoss(NamedTuple):
    """``loss``: scalar; ``logp``: ``[n]`` summed log-probabilities of the sequences under the policy (differentiable, so a
    likelihood term can be added); ``ref_logp``: ``[n]`` the same under the reference (zeros without one), a constant."""
    loss: torch.Tensor
    logp: torch.Tensor
    ref_logp: torch.Tensor


class PolicyLoss(NamedTuple):
    """``loss``: scalar; ``logp``: ``[n, s]`` log-probabilities of the labels, zero where the mask is; ``kl`` and ``clipped``:
    mean KL estimate and share of clipped tokens over the mask.  All but ``loss`` are constants."""
    loss: torch.Tensor
    logp: torch.Tensor
    kl: torch.Tensor
    clipped: torch.Tensor


# ---------------------------------------------------------------------------------------------- arguments
def _constant(name, t):
    if t is not None and t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} is a constant of this loss and gets no gradient: detach it")
    return t


def _check(logits, labels, loss_mask, ref_logits, ref_logp):
    if logits.dim() != 3 or logits.shape[0] == 0 or logits.shape[2] == 0:
        raise ValueError(f"logits are [sequences, tokens, vocabulary] of at least one sequence and word, got {tuple(logits.shape)}")
    if not logits.is_floating_point():
        raise ValueError(f"logits are floating-point numbers, got {logits.dtype}")
    for name, t in (("labels", labels), ("loss_mask", loss_mask), ("ref_logp", ref_logp)):
        if t is not None and t.shape != logits.shape[:2]:
            raise ValueError(f"{name} is {tuple(t.shape)}, the logits' sequences are {tuple(logits.shape[:2])}")
    if labels.is_floating_point() or labels.dtype == torch.bool:
        raise ValueError(f"labels are integers, got {labels.dtype}")
    if ref_logits is not None:
        if ref_logp is not None:
            raise ValueError("give ref_logits or ref_logp, not both")
        if ref_logits.shape != logits.shape or ref_logits.dtype != logits.dtype:
            raise ValueError(f"ref_logits are {tuple(ref_logits.shape)} {ref_logits.dtype}, logits {tuple(logits.shape)} "
                             f"{logits.dtype}")
    for name, t in (("loss_mask", loss_mask), ("ref_logits", ref_logits), ("ref_logp", ref_logp)):
        _constant(name, t)
    for name, t in (("labels", labels), ("loss_mask", loss_mask), ("ref_logits", ref_logits), ("ref_logp", ref_logp)):
        if t is not None and t.device != logits.device:
            raise ValueError(f"{name} is on {t.device}, the logits are on {logits.device}")


def _as(t, dtype):
    """A constant as the kernels read it: contiguous, of that type."""
    if t is None or (t.dtype == dtype and t.is_contiguous()):
        return t
    return t.to(dtype).contiguous()


def _rows(t):
    """Logits whose vocabulary is contiguous; batch and time may have any strides."""
    return t if t is None or t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _tensor_parallel():
    from ..parallel import mpu
    return mpu.get_model_parallel_world_size(), mpu.get_model_parallel_rank(), mpu.get_model_parallel_group


# ---------------------------------------------------------------------------------------------- kernels
class _Stats:
    """One pass over the kept rows of policy (and reference) logits, and the scratch memory of a forward, in one piece::

        sums    [n * (pieces + 1), width] fp64    what the joining kernel's blocks leave
        part    [streams, rows, most, 2]          maximum and sum of every chunk of a row, policy and reference
        cross   [rows, most]                      sum of p (x - y), for the KL over the vocabulary
        target  [streams, rows]                   the labels' logits
        ticket  [2] int32

    With the vocabulary split over ranks the chunks are joined here and two all-reduces -- maxima, then sums and label logits --
    make the statistics those of whole rows.  What stands in rows of mask zero is never read."""

    def __init__(self, x, y, labels, mask, full, width):
        n, s, v = x.shape
        rows = n * s
        streams = 1 if y is None else 2
        tp, rank, group = _tensor_parallel()
        L, dt = native.lib(), _DT[x.dtype]
        most = L.neox_vocab_splits(rows, v, dt, full)
        sums = 2 * width * n * (L.neox_loss_pieces(s) + 1)
        parts = streams * rows * most * 2
        crosses = rows * most if full else 0
        self.buf = buf = torch.empty(sums + parts + crosses + streams * rows + 2, dtype=torch.float32, device=x.device)
        self.sums = buf.data_ptr()
        self.part = self.sums + 4 * sums
        self.cross = self.part + 4 * parts
        self.target = self.cross + 4 * crosses
        self.ticket = self.target + 4 * streams * rows
        self.most, self.chunks, self.first, self.vocab = most, 0, rank * v, tp * v
        y_ = x if y is None else y
        rc = L.neox_vocab_stats(x.data_ptr(), x.stride(0), x.stride(1), None if y is None else y.data_ptr(), y_.stride(0),
                                y_.stride(1), labels.data_ptr(), mask.data_ptr(), n, s, v, self.first, dt, full, self.part,
                                self.cross, self.target, self.ticket, native.stream_ptr())
        native.check(rc, "neox_vocab_stats")
        if tp > 1:
            self._reduce(sums, parts, crosses, streams, rows, group())

    def _reduce(self, sums, parts, crosses, streams, rows, group):
        import torch.distributed as dist
        _, part, cross, target, ticket = self.buf.split([sums, parts, crosses, streams * rows, 2])
        part, target = part.view(streams, rows, self.most, 2), target.view(streams, rows)
        there = torch.arange(self.most, device=part.device) < ticket.view(torch.int32)[1]
        local = torch.where(there, part[..., 0], torch.finfo(torch.float32).min)
        top = local.amax(-1)
        dist.all_reduce(top, op=dist.ReduceOp.MAX, group=group)
        scale = (local - top[..., None]).exp()
        terms = [torch.where(there, part[..., 1] * scale, 0.0).sum(-1), target]
        if crosses:
            terms.append(torch.where(there, cross.view(rows, self.most) * scale[0], 0.0).sum(-1)[None])
        both = torch.cat(terms)
        dist.all_reduce(both, group=group)
        joined = torch.stack([top, both[:streams]], -1)
        self.keep = (joined, both)
        self.part, self.target = joined.data_ptr(), both[streams].data_ptr()
        self.cross = both[-1].data_ptr() if crosses else 0
        self.most = self.chunks = 1


def _logits_grad(x, y, labels, slope, mask, shift, row, coef, g_loss, g_logp, kl_beta, first):
    """Gradient of the logits in their own memory order where that is dense.  ``slope`` to ``coef`` are addresses."""
    n, s, v = x.shape
    g = torch.empty_like(x)
    if g.stride(2) != 1:
        g = torch.empty(n, s, v, dtype=x.dtype, device=x.device)
    y_ = x if y is None else y
    rc = native.lib().neox_vocab_grad(
        x.data_ptr(), x.stride(0), x.stride(1), y_.data_ptr(), y_.stride(0), y_.stride(1), g.data_ptr(), g.stride(0), g.stride(1),
        labels.data_ptr(), slope, mask.data_ptr(), shift, row, coef, None if g_loss is None else g_loss.data_ptr(),
        None if g_logp is None else g_logp.data_ptr(), kl_beta, n, s, v, first, _DT[x.dtype], native.stream_ptr())
    native.check(rc, "neox_vocab_grad")
    return g


def _preference_values(x, labels, mask, ref_logits, ref_logp, beta, smoothing):
    """Loss, log-probabilities, what the backward needs (``[rows, 2]`` maximum and 1 / sum, then ``[n]`` coefficients), and the
    first word of this rank's vocabulary."""
    n, s, _ = x.shape
    st = _Stats(x, ref_logits, labels, mask, 0, 2)
    dev = x.device
    kept = torch.empty(2 * n * s + n, dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    logp = torch.empty(n, dtype=torch.float32, device=dev)
    ref = torch.empty(n, dtype=torch.float32, device=dev)
    row = kept.data_ptr()
    rc = native.lib().neox_preference_loss(
        st.part, st.target, st.most, st.chunks, labels.data_ptr(), mask.data_ptr(), None if ref_logp is None else ref_logp.data_ptr(),
        ref_logits is not None, n, s, st.vocab, beta, smoothing, row, st.sums, st.ticket, loss.data_ptr(), logp.data_ptr(),
        ref.data_ptr(), row + 8 * n * s, native.stream_ptr())
    native.check(rc, "neox_preference_loss")
    return loss, logp, ref, kept, st.first


def _grad_f32(g):
    return None if g is None else _as(g, torch.float32)


class _PreferenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, labels, mask, ref_logits, ref_logp, beta, smoothing):
        with device_of(x):
            loss, logp, ref, kept, ctx.first = _preference_values(x, labels, mask, ref_logits, ref_logp, beta, smoothing)
        ctx.save_for_backward(x, labels, mask, kept)
        ctx.mark_non_differentiable(ref)
        ctx.set_materialize_grads(False)
        return loss, logp, ref

    @staticmethod
    def backward(ctx, g_loss, g_logp, _):
        x, labels, mask, kept = ctx.saved_tensors
        if g_loss is None and g_logp is None:
            return (None,) * 7
        row = kept.data_ptr()
        with device_of(x):
            g = _logits_grad(x, None, labels, mask.data_ptr(), mask, None, row, row + 8 * mask.numel(), _grad_f32(g_loss),
                             _grad_f32(g_logp), 0.0, ctx.first)
        return (once(g, x),) + (None,) * 6


def _policy_values(x, labels, mask, adv, old_logp, ref_logits, ref_logp, low, high, kl, kl_beta, by_sequence):
    """Loss, means, log-probabilities, what the backward needs (``[rows, 2]`` maximum and 1 / sum, ``[n]`` coefficients, ``[rows]``
    slopes and, for the KL over the vocabulary, ``[rows]`` shifts), and the first word of this rank's vocabulary."""
    n, s, _ = x.shape
    rows, full = n * s, kl == KL_KINDS["full"]
    st = _Stats(x, ref_logits, labels, mask, int(full), 4)
    dev = x.device
    kept = torch.empty((4 if full else 3) * rows + n, dtype=torch.float32, device=dev)
    out = torch.empty(3, dtype=torch.float32, device=dev)
    logp = torch.empty(n, s, dtype=torch.float32, device=dev)
    row = kept.data_ptr()
    coef = row + 8 * rows
    slope = coef + 4 * n
    rc = native.lib().neox_policy_loss(
        st.part, st.cross, st.target, st.most, st.chunks, labels.data_ptr(), mask.data_ptr(), adv.data_ptr(), adv.stride(0),
        adv.stride(1), None if old_logp is None else old_logp.data_ptr(), None if ref_logp is None else ref_logp.data_ptr(),
        ref_logits is not None, n, s, st.vocab, kl, by_sequence, low, high, kl_beta, row, slope, slope + 4 * rows if full else None,
        st.sums, st.ticket, out.data_ptr(), logp.data_ptr(), coef, native.stream_ptr())
    native.check(rc, "neox_policy_loss")
    return (*out.unbind(0), logp, kept, st.first)


class _PolicyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, labels, mask, adv, old_logp, ref_logits, ref_logp, low, high, kl, kl_beta, by_sequence):
        with device_of(x):
            loss, mean_kl, clipped, logp, kept, ctx.first = _policy_values(x, labels, mask, adv, old_logp, ref_logits, ref_logp, low,
                                                                           high, kl, kl_beta, by_sequence)
        ctx.full, ctx.kl_beta = kl == KL_KINDS["full"], kl_beta
        ctx.save_for_backward(x, labels, mask, kept, ref_logits if ctx.full else None)
        ctx.mark_non_differentiable(mean_kl, clipped, logp)
        ctx.set_materialize_grads(False)
        return loss, mean_kl, clipped, logp

    @staticmethod
    def backward(ctx, g_loss, *_):
        x, labels, mask, kept, ref_logits = ctx.saved_tensors
        if g_loss is None:
            return (None,) * 12
        rows, row = mask.numel(), kept.data_ptr()
        coef = row + 8 * rows
        slope = coef + 4 * mask.shape[0]
        with device_of(x):
            g = _logits_grad(x, ref_logits, labels, slope, mask, slope + 4 * rows if ctx.full else None, row, coef,
                             _grad_f32(g_loss), None, ctx.kl_beta, ctx.first)
        return (once(g, x),) + (None,) * 11


# ---------------------------------------------------------------------------------------------- plain statements
def _kept_logits(logits, loss_mask):
    return logits.masked_fill((loss_mask == 0).unsqueeze(-1), 0.0)


def _label_logp(logits, labels, loss_mask):
    """Log-probabilities of the labels in 32 bits (64 for 64-bit logits); what stands at masked positions does not matter."""
    labels = torch.where(loss_mask == 0, torch.zeros_like(labels), labels).long()
    logits = _kept_logits(logits, loss_mask)
    tp = _tensor_parallel()[0]
    if tp > 1:
        from ..parallel.cross_entropy import vocab_parallel_cross_entropy
        logp, vocab = -vocab_parallel_cross_entropy(logits.float(), labels), tp * logits.shape[-1]
    else:
        wide = logits if logits.dtype == torch.float64 else logits.float()
        vocab = logits.shape[-1]
        logp = wide.log_softmax(-1).gather(-1, labels.clamp(0, vocab - 1)[..., None])[..., 0]
    return torch.where((labels < 0) | (labels >= vocab), torch.full_like(logp, float("nan")), logp)


def _value_type(logits):
    return torch.float64 if logits.dtype == torch.float64 else torch.float32


def preference_loss_ref(logits, labels, loss_mask, beta, ref_logits=None, ref_logp=None, label_smoothing=0.0):
    """:func:`preference_loss` in plain PyTorch."""
    def summed(logp):
        return torch.where(loss_mask == 0, torch.zeros_like(logp), logp * loss_mask).double().sum(-1)

    logp = summed(_label_logp(logits, labels, loss_mask))
    with torch.no_grad():
        if ref_logits is not None:
            ref = summed(_label_logp(ref_logits, labels, loss_mask))
        else:
            ref = summed(ref_logp) if ref_logp is not None else torch.zeros_like(logp)
    margin = logp - ref
    chosen, rejected = margin.chunk(2)
    z = beta * (chosen - rejected)
    loss = -(1 - label_smoothing) * F.logsigmoid(z)
    if label_smoothing:
        loss = loss - label_smoothing * F.logsigmoid(-z)
    dt = _value_type(logits)
    return PreferenceLoss(loss.mean().to(dt), logp.to(dt), ref.to(dt))


def policy_loss_ref(logits, labels, loss_mask, advantages, old_logp=None, ref_logits=None, ref_logp=None, clip_low=0.2,
                    clip_high=None, kl="k3", kl_beta=0.0, reduce="token"):
    """:func:`policy_loss` in plain PyTorch."""
    clip_high = clip_low if clip_high is None else clip_high
    keep = loss_mask != 0
    zero = lambda t: torch.where(keep, t, torch.zeros_like(t))          # noqa: E731
    logp = _label_logp(logits, labels, loss_mask).double()
    adv = zero((advantages if advantages.dim() == 2 else advantages[:, None]).expand(logp.shape).double())
    old = logp.detach() if old_logp is None else zero(old_logp.double())
    ratio = (zero(logp) - zero(old)).exp()
    free, held = ratio * adv, ratio.clamp(1 - clip_low, 1 + clip_high) * adv
    clipped = free > held
    term = -torch.where(clipped, held.detach(), free)
    if kl == "full":
        x, y = _kept_logits(logits, loss_mask), _kept_logits(ref_logits.detach(), loss_mask)
        if _tensor_parallel()[0] > 1:
            from ..parallel import mappings as M
            x, y = M.gather_from_model_parallel_region(x), M.gather_from_model_parallel_region(y)
        dt = _value_type(x)
        lx, ly = x.to(dt).log_softmax(-1), y.to(dt).log_softmax(-1)
        impossible = x == -float("inf")                                 # probability zero adds nothing
        each = (lx.masked_fill(impossible, 0.0) - ly.masked_fill(impossible, 0.0)) * lx.exp()
        estimate = each.double().sum(-1)
    elif ref_logits is not None or ref_logp is not None:
        with torch.no_grad():
            ref = _label_logp(ref_logits, labels, loss_mask) if ref_logits is not None else ref_logp
        d = zero(logp) - zero(ref.double())
        estimate = {"kl": lambda: d, "abs": d.abs, "mse": lambda: 0.5 * d.square(), "k3": lambda: torch.expm1(-d) + d}[kl]()
    else:
        estimate = torch.zeros_like(logp)
    w = loss_mask.double()
    length = w.sum(-1)
    total = length.sum()
    mean = lambda t: torch.where(total != 0, (zero(t) * w).sum() / total, torch.zeros_like(total))     # noqa: E731
    term = zero(term + kl_beta * estimate) * w
    if reduce == "token":
        loss = term.sum() / torch.where(total != 0, total, torch.ones_like(total))
    else:
        filled = length > 0
        loss = torch.where(filled, term.sum(-1) / torch.where(filled, length, torch.ones_like(length)), 0.0).sum()
        loss = loss / filled.sum().clamp(min=1)
    dt = _value_type(logits)
    return PolicyLoss(loss.to(dt), zero(logp).detach().to(dt), mean(estimate).detach().to(dt),
                      mean(clipped.double()).detach().to(dt))


# ---------------------------------------------------------------------------------------------- entry points
def preference_loss(logits, labels, loss_mask, beta, ref_logits: Optional[torch.Tensor] = None,
                    ref_logp: Optional[torch.Tensor] = None, label_smoothing: float = 0.0) -> PreferenceLoss:
    """Preference loss over the pairs (sequence ``i``, sequence ``n / 2 + i``) of a batch ``[chosen; rejected]``::

        z = beta * ((logp_chosen - logp_rejected) - (ref_chosen - ref_rejected))
        loss = mean(-(1 - e) * log sigmoid(z) - e * log sigmoid(-z)),      e = label_smoothing

    ``logits``: ``[n, s, V / tp]`` (bf16, fp16 or fp32, any strides with a contiguous vocabulary); ``labels``: ``[n, s]`` over the
    whole vocabulary, one outside makes its pair NaN; ``loss_mask``: ``[n, s]``, the weight of every position.  The reference is
    ``ref_logits`` (shape and type of ``logits``), ``ref_logp`` (``[n, s]``) or nothing.  Reference and mask are constants.  A
    sequence without a kept position has log-probability zero.  The gradient can be taken once, not differentiated again.
    """
    _check(logits, labels, loss_mask, ref_logits, ref_logp)
    if logits.shape[0] % 2:
        raise ValueError(f"pairs are [chosen; rejected]: an even number of sequences, got {logits.shape[0]}")
    if not 0.0 <= label_smoothing < 1.0:
        raise ValueError(f"label_smoothing is at least 0 and below 1, got {label_smoothing}")
    if not _k(logits):
        return preference_loss_ref(logits, labels, loss_mask, beta, ref_logits, ref_logp, label_smoothing)
    args = (_rows(logits), _as(labels, torch.int64), _as(loss_mask, torch.float32), _rows(ref_logits),
            _as(ref_logp, torch.float32), float(beta), float(label_smoothing))
    if native.plain_call(logits):
        with device_of(logits):
            return PreferenceLoss(*_preference_values(*args)[:3])
    return PreferenceLoss(*_PreferenceFn.apply(*args))


def policy_loss(logits, labels, loss_mask, advantages, old_logp: Optional[torch.Tensor] = None,
                ref_logits: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, clip_low: float = 0.2,
                clip_high: Optional[float] = None, kl: str = "k3", kl_beta: float = 0.0, reduce: str = "token") -> PolicyLoss:
    """Clipped policy loss with a KL term.  With ``l`` the log-probability of a label, ``A`` its advantage::

        r = exp(l - old_logp)                                      (1 without old_logp: the policy that sampled is the present one)
        term = -min(r * A, clip(r, 1 - clip_low, 1 + clip_high) * A) + kl_beta * KL

    ``kl`` names the estimate, with ``d = l - l_ref``: ``"kl"`` d, ``"abs"`` |d|, ``"mse"`` d^2 / 2, ``"k3"`` exp(-d) - 1 + d, or
    ``"full"``: the KL from policy to reference over the whole vocabulary, which needs ``ref_logits``.  Without a reference there
    is no KL term.  ``reduce``: ``"token"``, the mean over all kept positions, weighted by ``loss_mask``; ``"sequence"``, the mean
    over the sequences that keep one of each sequence's own mean.  Nothing kept: loss and gradient are zero.

    ``logits``, ``labels``, ``loss_mask``, ``ref_logits``, ``ref_logp`` as in :func:`preference_loss`; ``advantages``: ``[n, s]``, or
    ``[n]`` for one a sequence; ``old_logp``: ``[n, s]``.  All but ``logits`` are constants.
    """
    _check(logits, labels, loss_mask, ref_logits, ref_logp)
    n, s = logits.shape[:2]
    clip_high = clip_low if clip_high is None else clip_high
    if advantages.dim() == 1:
        advantages = advantages[:, None]
    if advantages.dim() != 2 or advantages.shape[0] not in (1, n) or advantages.shape[1] not in (1, s):
        raise ValueError(f"advantages are [{n}, {s}] or [{n}], got {tuple(advantages.shape)}")
    if old_logp is not None and old_logp.shape != labels.shape:
        raise ValueError(f"old_logp is {tuple(old_logp.shape)}, the logits' sequences are {(n, s)}")
    for name, t in (("advantages", advantages), ("old_logp", old_logp)):
        if t is not None and t.device != logits.device:
            raise ValueError(f"{name} is on {t.device}, the logits are on {logits.device}")
        _constant(name, t)
    if kl not in KL_KINDS:
        raise ValueError(f"kl is one of {', '.join(KL_KINDS)}, got {kl!r}")
    if kl == "full" and ref_logits is None:
        raise ValueError("the KL over the whole vocabulary needs ref_logits")
    if reduce not in ("token", "sequence"):
        raise ValueError(f"reduce is token or sequence, got {reduce!r}")
    if not (0.0 <= clip_low <= 1.0 and clip_high >= 0.0):
        raise ValueError(f"the ratio is clipped to [1 - clip_low, 1 + clip_high] with clip_low in [0, 1] and clip_high >= 0, got "
                         f"{clip_low} and {clip_high}")
    if not _k(logits):
        return policy_loss_ref(logits, labels, loss_mask, advantages, old_logp, ref_logits, ref_logp, clip_low, clip_high, kl,
                               kl_beta, reduce)
    if advantages.dtype != torch.float32:
        advantages = advantages.to(torch.float32)
    kind = KL_KINDS[kl] if ref_logits is not None or ref_logp is not None else 0
    args = (_rows(logits), _as(labels, torch.int64), _as(loss_mask, torch.float32), advantages.expand(n, s),
            _as(old_logp, torch.float32), _rows(ref_logits), _as(ref_logp, torch.float32), 1.0 - clip_low, 1.0 + clip_high, kind,
            float(kl_beta), reduce == "sequence")
    if native.plain_call(logits):
        with device_of(logits):
            loss, mean_kl, clipped, logp = _policy_values(*args)[:4]
    else:
        loss, mean_kl, clipped, logp = _PolicyFn.apply(*args)
    return PolicyLoss(loss, logp, mean_kl, clipped)
