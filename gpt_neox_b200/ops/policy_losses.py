"""Losses of post-training on vocabulary-parallel logits: a preference loss over pairs of sequences and a clipped policy loss
with a KL term.

Both are functions of the log-probabilities that a policy gives the labels of the positions whose ``loss_mask`` is not zero.
Positions of mask zero -- prompts, padding -- are not read: their logits may hold anything and their gradient is zero.  On a GPU
the logits are streamed once for the loss and once for its gradient -- a policy loss writes both from one reading where it can --
(``csrc/policy_losses.cu``), in their own type and memory order.  Exponentials and a lane's sums of them are in 32 bits; a row's
log-probability, the sums over a sequence, the ratios, z and the loss are in 64; coefficients of the gradient and outputs are
rounded to 32.  (Over a split vocabulary the ranks' sums are joined in 32 bits.)
``*_ref`` are the same losses in plain PyTorch: the CPU path and the statement the kernels are tested against.

Reference counterparts: the DPO and REINFORCE objectives of ``megatron/training.py:533-939``, which form ``[b, s, V]``
log-probabilities in fp32.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F

from . import native
from .functional import _DT, _k, device_of, once

KL_KINDS = {"kl": 1, "abs": 2, "mse": 3, "k3": 4, "full": 5}

native._ARGTYPES.update({
    "neox_vocab_chunks": [ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_int],
    "neox_loss_pieces": [ctypes.c_int],
    "neox_loss_forward": [ctypes.c_char_p],
    "neox_policy_fits": [ctypes.c_int, ctypes.c_int],
    "neox_policy_at_once": [ctypes.c_char_p],
    "neox_loss_backward": [ctypes.c_char_p],
})
native._CountingLib._NOT_LAUNCHES.update({"neox_vocab_chunks", "neox_loss_pieces", "neox_policy_fits"})

_MOST_TOKENS = _MOST_WORDS = 1 << 30    # the kernels number them, and steps past the last one, in 32 bits

# The kernels' arguments in the order of LossCall (csrc/policy_losses.cu): addresses and 64-bit words, doubles, ints.
_CALL = struct.Struct("@36q5d12i")


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
    if isinstance(t, torch.Tensor) and t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} is a constant of this loss and gets no gradient: detach it")
    return t


def _check(logits, labels, loss_mask, ref_logits, ref_logp):
    if logits.dim() != 3 or logits.shape[0] == 0 or logits.shape[2] == 0:
        raise ValueError(f"logits are [sequences, tokens, vocabulary] of at least one sequence and word, got {tuple(logits.shape)}")
    if not logits.is_floating_point():
        raise ValueError(f"logits are floating-point numbers, got {logits.dtype}")
    if logits.shape[0] * logits.shape[1] >= _MOST_TOKENS:
        raise ValueError(f"a batch has fewer than {_MOST_TOKENS} tokens, got {tuple(logits.shape)}")
    if logits.shape[2] >= _MOST_WORDS:
        raise ValueError(f"a vocabulary, or a rank's share of it, has fewer than {_MOST_WORDS} words, got {logits.shape[2]}")
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


@functools.lru_cache(maxsize=1)
def _mpu():
    from ..parallel import mpu                  # which imports this package
    return mpu


def _tensor_parallel():
    mpu = _mpu()
    return mpu.get_model_parallel_world_size(), mpu.get_model_parallel_rank(), mpu.get_model_parallel_group


# ---------------------------------------------------------------------------------------------- kernels
@functools.lru_cache(maxsize=256)
def _layout(n, s, v, dtype, streams, width, full, device):
    """Chunks of a row, and where the parts of a forward's one buffer begin, in bytes, with its size in floats at the end::

        sums    [n * (pieces + 1), width] fp64    what the joining kernel's blocks leave
        part    [streams, rows, most, 4]          of every chunk of a row, policy and reference: sum in 64 bits, maximum and, for the
                                                  KL over the vocabulary, sum of p (x - y)
        target  [streams, rows]                   the labels' logits
        ticket  [2] int32
        row     [rows, 2]                         maximum and 1 / sum, from here on kept for the backward
        coef    [n]
        slope   [rows]                            of the policy loss
        shift   [rows]                            for the KL over the vocabulary
    """
    L, rows = native.lib(), n * s
    most = L.neox_vocab_chunks(rows, v, dtype, full)
    sizes = (2 * width * n * (L.neox_loss_pieces(s) + 1), 4 * streams * rows * most, streams * rows, 2,
             2 * rows, n, rows * (width == 4), rows * full)
    at, offsets = 0, []
    for size in sizes:
        offsets.append(4 * at)
        at += size + size % 2                   # pairs of floats and doubles are read in one piece
    return (most, *offsets, at)


def _reduced(buf, at, streams, rows, most, full, group):
    """Statistics of whole rows from those of every rank's share of the vocabulary: the chunks are joined here and two all-reduces
    follow, maxima, then sums and label logits.  What stands in rows of mask zero is never read."""
    import torch.distributed as dist
    _, part, target, ticket = (o // 4 for o in at[:4])
    part = buf[part:part + 4 * streams * rows * most].view(streams, rows, most, 4)
    there = torch.arange(most, device=buf.device) < buf[ticket:ticket + 2].view(torch.int32)[1]
    local = torch.where(there, part[..., 2], torch.finfo(torch.float32).min)
    top = local.amax(-1)
    dist.all_reduce(top, op=dist.ReduceOp.MAX, group=group)
    scale = (local - top[..., None]).exp()
    terms = [torch.where(there, part.view(torch.float64)[..., 0] * scale, 0.0).sum(-1).float(),
             buf[target:target + (1 if full else streams) * rows].view(-1, rows)]
    if full:
        terms.append(torch.where(there, part[0, ..., 3] * scale[0], 0.0).sum(-1)[None])
    both = torch.cat(terms)
    dist.all_reduce(both, group=group)
    whole = torch.empty(streams, rows, 4, dtype=torch.float32, device=buf.device)
    whole.view(torch.float64)[..., 0] = both[:streams]
    whole[..., 2] = top
    if full:
        whole[0, :, 3] = both[-1]
    return whole, both[streams:]


def _forward(x, y, labels, mask, width, loss, kl_mean, clipped, logp, ref, old_logp, ref_logp, adv, kl, by_sequence, beta, smoothing,
             low, high, wide=None):
    """Runs a forward into the given outputs; the buffer whose end the backward needs, and the first word of this rank's share of
    the vocabulary."""
    n, s, v = x.shape
    dt, streams, full = _DT[x.dtype], 1 if y is None else 2, int(kl == KL_KINDS["full"])
    tp, rank, group = _tensor_parallel()
    most, *at, total = _layout(n, s, v, dt, streams, width, full, x.get_device())
    buf = torch.empty(total, dtype=torch.float32, device=x.device)
    base = buf.data_ptr()
    sums, part, target, ticket, row, coef, slope, shift = [base + o for o in at]
    y_ = x if y is None else y
    head = (x.data_ptr(), x.stride(0), x.stride(1), 0 if y is None else y.data_ptr(), y_.stride(0), y_.stride(1),
            labels.data_ptr(), mask.data_ptr())
    tail = (ticket, sums, row, coef, slope, shift if full else 0, loss.data_ptr(), 0 if kl_mean is None else kl_mean.data_ptr(),
            0 if clipped is None else clipped.data_ptr(), logp.data_ptr(), 0 if ref is None else ref.data_ptr(),
            0 if old_logp is None else old_logp.data_ptr(), 0 if ref_logp is None else ref_logp.data_ptr(),
            *((0, 0, 0) if adv is None else (adv.data_ptr(), adv.stride(0) if adv.shape[0] > 1 else 0,
                                             adv.stride(1) if adv.shape[1] > 1 else 0)),
            0, 0, 0, 0, 0, rank * v, tp * v, native.stream_ptr(), 0, 0 if wide is None else wide.data_ptr(), beta, smoothing, low, high, 0.0,
            n, s, v, dt, kl, by_sequence)
    run = native.lib().neox_loss_forward
    policy = width == 4
    if tp == 1:
        native.check(run(_CALL.pack(*head, part, target, *tail, most, 0, policy, 1, 1, 0)), "neox_loss_forward")
    else:
        native.check(run(_CALL.pack(*head, part, target, *tail, most, 0, policy, 1, 0, 0)), "neox_loss_forward")
        whole, targets = _reduced(buf, at, streams, n * s, most, full, group())
        native.check(run(_CALL.pack(*head, whole.data_ptr(), targets.data_ptr(), *tail, 1, 1, policy, 0, 1, 0)),
                     "neox_loss_forward")
    return buf, rank * v


def _new_grad(x):
    """A gradient whose rows lie as the logits' do, so that both are read and written 16 bytes at a time: logits without their last
    position or without padding words leave the same gaps in it, as long as it is half full."""
    n, s, v = x.shape
    if x.is_contiguous() and not x.data_ptr() & 15:
        return torch.empty_like(x)
    (a, size_a), (b, size_b) = sorted(((x.stride(0), n), (x.stride(1), s)))
    inner = a * (size_a - 1) + v
    span = b * (size_b - 1) + inner
    if (size_a > 1 and a < v) or (size_b > 1 and b < inner) or span > 2 * x.numel():
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    shift = (x.data_ptr() & 15) // x.element_size()
    return torch.empty(shift + span, dtype=x.dtype, device=x.device).as_strided(x.shape, x.stride(), shift)


def _backward(x, y, labels, mask, g, row, coef, slope, shift, first, g_loss, g_logp, beta, expected, done):
    """Writes the gradient of the logits into ``g``.  ``y``: the reference, for the KL over the vocabulary; ``row`` to ``shift``:
    addresses of what the forward kept; ``done``: ``g`` is already right if the gradient of the loss is ``expected``."""
    n, s, v = x.shape
    y_ = x if y is None else y
    call = _CALL.pack(x.data_ptr(), x.stride(0), x.stride(1), y_.data_ptr(), y_.stride(0), y_.stride(1), labels.data_ptr(),
                      mask.data_ptr(), 0, 0, 0, 0, row, coef, slope, shift, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, g.data_ptr(), g.stride(0),
                      g.stride(1), 0 if g_loss is None else g_loss.data_ptr(), 0 if g_logp is None else g_logp.data_ptr(), first, 0,
                      native.stream_ptr(), 0, 0, beta, 0.0, 0.0, 0.0, expected, n, s, v, _DT[x.dtype], 0, 0, 0, 0, 0, 0, 0, done)
    native.check(native.lib().neox_loss_backward(call), "neox_loss_backward")
    return g


def _kept(x, buf, streams, width, full):
    """Addresses of what a forward kept in its buffer: row statistics, coefficients, slopes, shifts."""
    n, s, v = x.shape
    at = _layout(n, s, v, _DT[x.dtype], streams, width, full, x.get_device())
    base = buf.data_ptr()
    return base + at[5], base + at[6], base + at[7], base + at[8] if full else 0


def _preference_values(x, labels, mask, ref_logits, ref_logp, beta, smoothing):
    n, dev = x.shape[0], x.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    logp = torch.empty(n, dtype=torch.float32, device=dev)
    ref = torch.empty(n, dtype=torch.float32, device=dev)
    kept = _forward(x, ref_logits, labels, mask, 2, loss, None, None, logp, ref, None, ref_logp, None, 0, 0, beta, smoothing, 0.0, 0.0)
    return loss, logp, ref, kept


def _grad_f32(g):
    return g if g is None or (g.dtype == torch.float32 and g.is_contiguous()) else g.float().contiguous()


class _PreferenceFn(torch.autograd.Function):
    """All but the logits are constants and come as one argument: autograd looks at each of them otherwise."""

    @staticmethod
    def forward(ctx, x, rest):
        labels, mask, ref_logits, ref_logp, beta, smoothing = rest
        with device_of(x):
            loss, logp, ref, (buf, ctx.first) = _preference_values(x, *rest)
        ctx.streams = 1 if ref_logits is None else 2
        ctx.save_for_backward(x, labels, mask, buf)
        ctx.mark_non_differentiable(ref)
        ctx.set_materialize_grads(False)
        return loss, logp, ref

    @staticmethod
    def backward(ctx, g_loss, g_logp, _):
        if g_loss is None and g_logp is None:
            return None, None
        x, labels, mask, buf = ctx.saved_tensors
        with device_of(x):
            row, coef, _, _ = _kept(x, buf, ctx.streams, 2, 0)
            g = _backward(x, None, labels, mask, _new_grad(x), row, coef, mask.data_ptr(), 0, ctx.first, _grad_f32(g_loss),
                          _grad_f32(g_logp), 0.0, 0.0, 0)
        return once(g, x), None


def _policy_values(x, labels, mask, adv, old_logp, ref_logits, ref_logp, low, high, kl, kl_beta, by_sequence, wide=None):
    dev = x.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    kl_mean = torch.empty((), dtype=torch.float32, device=dev)
    clipped = torch.empty((), dtype=torch.float32, device=dev)
    logp = torch.empty(x.shape[:2], dtype=torch.float32, device=dev)
    kept = _forward(x, ref_logits, labels, mask, 4, loss, kl_mean, clipped, logp, None, old_logp, ref_logp, adv, kl, by_sequence, kl_beta,
                    0.0, low, high, wide)
    return loss, kl_mean, clipped, logp, kept


@functools.lru_cache(maxsize=256)
def _at_once_layout(n, s):
    """As :func:`_layout`, for :func:`_policy_at_once`: ``row``, ``coef``, ``slope`` as there; of scratch, 4 fp64 for each of
    at most 2048 blocks, ``[n]`` fp64 and ``[rows + 2]`` int32."""
    rows = n * s
    sizes = (8 * min(rows, 2048), 2 * n, rows + 2, 2 * rows, n, rows)
    at, offsets = 0, []
    for size in sizes:
        offsets.append(4 * at)
        at += size + size % 2
    terms, _, _, row, coef, slope = offsets
    return row, coef, slope, terms, at


def _policy_at_once(x, labels, mask, adv, old_logp, ref_logp, wide, low, high, kl, kl_beta, by_sequence, expected):
    """The policy loss and, from the same reading of the logits, its gradient for a gradient ``expected`` of the loss.  ``wide``: the
    reference's log-probabilities in 64 bits, in place of ``ref_logp``."""
    n, s, v = x.shape
    dev = x.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    kl_mean = torch.empty((), dtype=torch.float32, device=dev)
    clipped = torch.empty((), dtype=torch.float32, device=dev)
    logp = torch.empty(n, s, dtype=torch.float32, device=dev)
    *at, total = _at_once_layout(n, s)
    buf = torch.empty(total, dtype=torch.float32, device=dev)
    row, coef, slope, terms = [buf.data_ptr() + o for o in at]
    g = _new_grad(x)
    call = _CALL.pack(x.data_ptr(), x.stride(0), x.stride(1), 0, 0, 0, labels.data_ptr(), mask.data_ptr(), 0, 0, 0, 0, row, coef,
                      slope, 0, loss.data_ptr(), kl_mean.data_ptr(), clipped.data_ptr(), logp.data_ptr(), 0,
                      0 if old_logp is None else old_logp.data_ptr(), 0 if ref_logp is None else ref_logp.data_ptr(),
                      adv.data_ptr(), adv.stride(0) if adv.shape[0] > 1 else 0, adv.stride(1) if adv.shape[1] > 1 else 0,
                      g.data_ptr(), g.stride(0), g.stride(1), 0, 0, 0, v, native.stream_ptr(), terms,
                      0 if wide is None else wide.data_ptr(), kl_beta, 0.0, low, high, expected, n, s, v, _DT[x.dtype], kl, by_sequence, 0, 0, 1, 0, 0, 1)
    native.check(native.lib().neox_policy_at_once(call), "neox_policy_at_once")
    return loss, kl_mean, clipped, logp, buf, g


# Bytes of logits from which on a reference's log-probabilities are taken first, in launches of their own, so that the policy's logits
# are read once: forward and backward of 8 x 1024 tokens over 50304 16-bit words (824 MB) 336 us so, 361 with both read together and
# the policy's twice; 4 x 4096 over 32064 (1 GB) 433 and 473; 4 x 512 over 50304 (206 MB) 116 and 118, but 30 us more for the host.
_REF_FIRST = 1 << 29
# Estimates whose references are always read together with the policy: the KL over the vocabulary, and |d|, whose slope jumps at d = 0,
# so that a policy equal to its reference -- the first step of training -- needs both log-probabilities from sums of the same order.
_TOGETHER = (KL_KINDS["full"], KL_KINDS["abs"])


@functools.lru_cache(maxsize=256)
def _one_reading_pays(vocab, dtype):
    """A row that keeps a block busy and fits in shared memory; others are read twice."""
    return vocab * dtype.itemsize >= 16384 and bool(native.lib().neox_policy_fits(vocab, _DT[dtype]))


class _PolicyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rest):
        labels, mask, adv, old_logp, ref_logits, ref_logp, low, high, kl, kl_beta, by_sequence, expected = rest
        # 16-bit floating-point numbers of five exponent bits need the loss scale before they are rounded
        at_once = ctx.needs_input_grad[0] and x.shape[1] > 0 and _tensor_parallel()[0] == 1 and (x.dtype != torch.float16 or expected != 1.0) \
            and (ref_logits is None or (kl not in _TOGETHER and x.numel() * x.element_size() >= _REF_FIRST)) \
            and _one_reading_pays(x.shape[2], x.dtype)
        ctx.full, ctx.kl_beta, ctx.expected, ctx.first, ctx.grad = int(kl == KL_KINDS["full"]), kl_beta, expected, 0, None
        with device_of(x):
            if at_once:
                wide = None
                if ref_logits is not None:
                    wide = torch.empty(x.shape[:2], dtype=torch.float64, device=x.device)
                    _policy_values(ref_logits, labels, mask, adv, None, None, None, low, high, 0, 0.0, False, wide)
                loss, kl_mean, clipped, logp, buf, ctx.grad = _policy_at_once(x, labels, mask, adv, old_logp, ref_logp, wide, low, high, kl,
                                                                              kl_beta, by_sequence, expected)
                ctx.streams, ctx.capture = 0, native.capture_id()
            else:
                loss, kl_mean, clipped, logp, (buf, ctx.first) = _policy_values(x, *rest[:-1])
                ctx.streams = 1 if ref_logits is None else 2
        ctx.save_for_backward(x, labels, mask, buf, ref_logits if ctx.full else None)
        ctx.mark_non_differentiable(kl_mean, clipped, logp)
        ctx.set_materialize_grads(False)
        return loss, kl_mean, clipped, logp

    @staticmethod
    def backward(ctx, g_loss, *_):
        if g_loss is None:
            return None, None
        x, labels, mask, buf, y = ctx.saved_tensors
        with device_of(x):
            # handed out once: a second backward through a retained graph writes another, as does one that is replayed without the
            # forward or the other way round, since a gradient may be changed by whoever got it
            done = ctx.grad is not None and native.capture_id() == ctx.capture
            g = None
            if done:
                g, ctx.grad = ctx.grad, None
            if ctx.streams:
                row, coef, slope, shift = _kept(x, buf, ctx.streams, 4, ctx.full)
            else:
                row, coef, slope = (buf.data_ptr() + o for o in _at_once_layout(x.shape[0], x.shape[1])[:3])
                shift = 0
            g = _backward(x, y, labels, mask, g if done else _new_grad(x), row, coef, slope, shift, ctx.first, _grad_f32(g_loss), None,
                          ctx.kl_beta, ctx.expected, done)
        return once(g, x), None


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
    ``ref_logits`` (shape and type of ``logits``), ``ref_logp`` (``[n, s]``) or nothing.  Reference, mask and numbers are constants.  A
    sequence without a kept position has log-probability zero.  The gradient can be taken once, not differentiated again.
    """
    _check(logits, labels, loss_mask, ref_logits, ref_logp)
    _constant("beta", beta)
    _constant("label_smoothing", label_smoothing)
    if logits.shape[0] % 2:
        raise ValueError(f"pairs are [chosen; rejected]: an even number of sequences, got {logits.shape[0]}")
    if not 0.0 <= label_smoothing < 1.0:
        raise ValueError(f"label_smoothing is at least 0 and below 1, got {label_smoothing}")
    if not _k(logits):
        return preference_loss_ref(logits, labels, loss_mask, beta, ref_logits, ref_logp, label_smoothing)
    x = _rows(logits)
    rest = (_as(labels, torch.int64), _as(loss_mask, torch.float32), _rows(ref_logits), _as(ref_logp, torch.float32), float(beta),
            float(label_smoothing))
    if native.plain_call(logits):
        with device_of(x):
            return PreferenceLoss(*_preference_values(x, *rest)[:3])
    return PreferenceLoss(*_PreferenceFn.apply(x, rest))


def policy_loss(logits, labels, loss_mask, advantages, old_logp: Optional[torch.Tensor] = None,
                ref_logits: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, clip_low: float = 0.2,
                clip_high: Optional[float] = None, kl: str = "k3", kl_beta: float = 0.0, reduce: str = "token",
                grad_scale: float = 1.0) -> PolicyLoss:
    """Clipped policy loss with a KL term.  With ``l`` the log-probability of a label, ``A`` its advantage::

        r = exp(l - old_logp)                                      (1 without old_logp: the policy that sampled is the present one)
        term = -min(r * A, clip(r, 1 - clip_low, 1 + clip_high) * A) + kl_beta * KL

    ``kl`` names the estimate, with ``d = l - l_ref``: ``"kl"`` d, ``"abs"`` |d|, ``"mse"`` d^2 / 2, ``"k3"`` exp(-d) - 1 + d, or
    ``"full"``: the KL from policy to reference over the whole vocabulary, which needs ``ref_logits``.  Without a reference there
    is no KL term.  ``reduce``: ``"token"``, the mean over all kept positions, weighted by ``loss_mask``; ``"sequence"``, the mean
    over the sequences that keep one of each sequence's own mean.  Nothing kept: loss and gradient are zero.

    ``logits``, ``labels``, ``loss_mask``, ``ref_logits``, ``ref_logp`` as in :func:`preference_loss`; ``advantages``: ``[n, s]``, or
    ``[n]`` for one a sequence; ``old_logp``: ``[n, s]``.  All but ``logits`` are constants.

    ``grad_scale`` is the gradient of the loss that the backward is expected to start from: 1 for ``loss.backward()``, a loss scale or
    ``1 / accumulation steps`` for a scaled loss.  Where the logits ask for a gradient, it is computed for that value together with
    the loss, while a row is at hand (its memory is taken then), and the backward only has to look; any other gradient of the loss
    is right as well, and costs the second reading of the logits that was to be saved.  (With the KL over the whole vocabulary, with
    fp16 logits and ``grad_scale`` 1, with reference logits in a small batch or for ``"abs"``, and for vocabularies that are short, split over ranks
    or too long for shared memory, logits are always read twice.)
    """
    _check(logits, labels, loss_mask, ref_logits, ref_logp)
    n, s = logits.shape[:2]
    for name, t in (("clip_low", clip_low), ("clip_high", clip_high), ("kl_beta", kl_beta)):
        _constant(name, t)
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
    x = _rows(logits)
    rest = (_as(labels, torch.int64), _as(loss_mask, torch.float32), advantages, _as(old_logp, torch.float32), _rows(ref_logits),
            _as(ref_logp, torch.float32), 1.0 - clip_low, 1.0 + clip_high, kind, float(kl_beta), reduce == "sequence", float(grad_scale))
    if native.plain_call(logits):
        with device_of(x):
            loss, mean_kl, clipped, logp = _policy_values(x, *rest[:-1])[:4]
    else:
        loss, mean_kl, clipped, logp = _PolicyFn.apply(x, rest)
    return PolicyLoss(loss, logp, mean_kl, clipped)
