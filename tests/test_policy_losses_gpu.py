"""Preference loss, clipped policy loss and the router with its losses on a GPU against their formulas in 64 bits.

Where the tolerances come from.  A kernel takes exp(x - max) in 32 bits with a fast exponential: a relative error of 2^-22 and,
for terms that count (x - max above -16), 2^-20 from the rounded argument; a thread adds some hundred of them to a running sum, whose
roundings (2^-24 each, of either sign) come to about 2^-20, the joins to a few more.  So a row's log-sum -- and with it a label's log-probability -- is off by at most 2^-18 =: ROW, and a
probability by that relative to itself.  All sums behind the rows are in 64 bits, results are rounded once to 32 bits (2^-24) or to
the type of the gradient (eps / 2 of it, and half of the smallest number of fp16, 2^-25; 32-bit numbers below 2^-126 are zero)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from gpt_neox_b200.ops import moe_ops as MO
from gpt_neox_b200.ops import policy_losses as PL

DEV = "cuda"
ROW = 2.0 ** -18


def _tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def _near(got, want, bound, what=""):
    got, want, bound = got.double(), want.double(), torch.as_tensor(bound, dtype=torch.float64, device=want.device).expand_as(want)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= bound)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, at {at} got {got[tuple(at)].item()!r}, want "
                             f"{want[tuple(at)].item()!r}, allowed {bound[tuple(at)].item()!r}")


def _logits(n, s, v, dtype, order="bsv", seed=0):
    """Logits like a model's, labels that stand out, in several memory orders."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, s, v, device=DEV, generator=g) * 2
    labels = torch.randint(0, v, (n, s), device=DEV, generator=g)
    x.scatter_add_(2, labels[..., None], torch.full((n, s, 1), 4.0, device=DEV))
    x = x.to(dtype)
    if order == "sbv":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    elif order == "shifted":                                  # rows that start off a 16-byte boundary
        x = torch.empty(n * s * v + 8, device=DEV, dtype=dtype)[1:1 + n * s * v].view(n, s, v).copy_(x)
    elif order == "padded":                                   # a slice of a wider vocabulary, later rows of a longer sequence
        wide = torch.full((n, s + 2, v + 5), 7.0, device=DEV, dtype=dtype)
        wide[:, 1:1 + s, :v] = x
        x = wide[:, 1:1 + s, :v]
    elif order == "strided":                                  # a vocabulary that is not contiguous
        x = torch.stack([x, x], -1)[..., 0]
    return x, labels


def _mask(n, s, seed, weights=False):
    g = torch.Generator(device=DEV).manual_seed(1000 + seed)
    m = (torch.rand(n, s, device=DEV, generator=g) > 0.4).float()
    if weights:
        m = m * (0.5 + torch.rand(n, s, device=DEV, generator=g))
    return m


def _row_bounds(x, labels, keep):
    """Probabilities and log-probabilities of the kept rows in 64 bits."""
    lp = x.double().log_softmax(-1)
    return lp.exp(), lp.gather(-1, labels[..., None])[..., 0], keep


SHAPES = [(2, 1, 1), (2, 3, 7), (4, 5, 64), (2, 9, 1000), (6, 2, 2049), (2, 4, 16385), (2, 3, 50257), (4, 300, 33), (2, 2, 130000)]


@pytest.mark.parametrize("order", ["bsv", "sbv", "shifted", "padded", "strided"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,s,v", SHAPES)
def test_preference_loss_matches_its_formula(n, s, v, dtype, order):
    seed = n * 7 + s * 3 + v
    x, labels = _logits(n, s, v, dtype, order, seed)
    mask = _mask(n, s, seed, weights=dtype == torch.float32)
    ref = {"bsv": "logits", "sbv": "logits", "shifted": "logp", "padded": None, "strided": "logits"}[order]
    ref_logits = (_logits(n, s, v, dtype, order, seed)[0] + torch.randn(n, s, v, device=DEV).to(dtype) * 0.3) if ref == "logits" else None
    ref_logp = -torch.rand(n, s, device=DEV) * 3 if ref == "logp" else None
    beta, eps, scale = 0.3, 0.1 if order == "sbv" else 0.0, 64.0
    x = x.detach().requires_grad_()
    out = PL.preference_loss(x, labels, mask, beta, ref_logits=ref_logits, ref_logp=ref_logp, label_smoothing=eps)
    g_loss, g_logp = torch.tensor(scale, device=DEV), torch.randn(n, device=DEV) * 0.1
    grad, = torch.autograd.grad([out.loss, out.logp], [x], [g_loss, g_logp])
    xd = x.detach().double().requires_grad_()
    want = PL.preference_loss_ref(xd, labels, mask.double(), beta, None if ref_logits is None else ref_logits.double(),
                                  None if ref_logp is None else ref_logp.double(), eps)
    want_grad, = torch.autograd.grad([want.loss, want.logp], [xd], [g_loss.double(), g_logp.double()])
    off = mask.double().sum(-1) * ROW
    _near(out.logp, want.logp.detach(), off + 2.0 ** -24 * want.logp.detach().abs(), "logp")
    _near(out.ref_logp, want.ref_logp, off + 2.0 ** -24 * want.ref_logp.abs(), "ref_logp")
    off_z = beta * 4 * off.max()                                   # four sums
    _near(out.loss, want.loss.detach(), off_z + 2.0 ** -24 * want.loss.detach().abs(), "loss")
    # a row's coefficient: the pair's slope (at most beta / pairs, its own slope in z at most a quarter of that) and g_logp
    coef = (scale * beta / (n // 2) + g_logp.abs().double())[:, None] * mask.double()
    off_coef = coef * (0.25 * off_z + 2.0 ** -21)
    p = xd.detach().softmax(-1)
    hot = torch.zeros_like(p).scatter_(-1, labels[..., None], 1.0)
    bound = torch.finfo(dtype).eps / 2 * want_grad.abs() + (off_coef[..., None] + 2.0 ** -20 * coef[..., None]) * (p + hot) \
        + 2 * ROW * coef[..., None] * p + _tiny(dtype)
    assert grad.dtype == dtype and grad.shape == x.shape
    _near(grad, want_grad, bound, "gradient")
    assert not grad[mask == 0].any()


@pytest.mark.parametrize("reduce", ["token", "sequence"])
@pytest.mark.parametrize("kl", ["none", "kl", "abs", "mse", "k3", "full"])
@pytest.mark.parametrize("n,s,v,dtype,order", [
    (1, 1, 9, torch.float32, "bsv"), (3, 5, 64, torch.bfloat16, "sbv"), (2, 300, 1031, torch.float16, "shifted"),
    (3, 4, 8200, torch.float32, "padded"), (2, 7, 50257, torch.bfloat16, "bsv"), (1, 6, 32000, torch.float16, "strided"),
    (5, 3, 1025, torch.bfloat16, "padded"), (2, 400, 8200, torch.bfloat16, "sbv"), (3, 70, 12001, torch.float32, "shifted"),
    (2, 90, 128256, torch.bfloat16, "bsv"), (40, 9, 9001, torch.float16, "padded"), (1100, 1, 8200, torch.bfloat16, "shifted"),
    (50, 70, 4099, torch.float32, "padded"), (2, 21, 100003, torch.bfloat16, "bsv"), (1, 3, 115711, torch.float16, "sbv"),
    (1, 3, 115712, torch.float16, "sbv"), (160, 2, 57856, torch.bfloat16, "shifted")])
def test_policy_loss_matches_its_formula(n, s, v, dtype, order, kl, reduce):
    seed = n * 11 + s + v
    x, labels = _logits(n, s, v, dtype, order, seed)
    mask = _mask(n, s, seed, weights=dtype == torch.float32)
    mask[0, 0] = 1.0
    if n > 2:
        mask[1] = 0.0                                              # a sequence that keeps nothing
    g = torch.Generator(device=DEV).manual_seed(seed)
    p, logp, _ = _row_bounds(x, labels, mask)
    # the sampler's log-probabilities: well inside or well outside of the clip's bounds, which are log 0.8 and log 1.3
    jump = torch.tensor([-0.6, -0.1, 0.0, 0.1, 0.6], device=DEV)[torch.randint(0, 5, (n, s), device=DEV, generator=g)]
    old = (logp - jump).float() if s != 4 else None
    adv = torch.randn(n, s, device=DEV, generator=g) if s != 7 else torch.randn(n, device=DEV, generator=g)
    noise = torch.randn(n, s, v, device=DEV, generator=g).to(dtype) * 0.3
    # from reference logits here and there, so that both ways are met
    ref_logits = (x + noise).as_strided(x.shape, (x + noise).stride()) if kl == "full" or (kl != "none" and s in (5, 6)) else None
    ref_logp = (logp + torch.where(jump > 0, 0.3, -0.2)).float() if kl != "none" and ref_logits is None else None
    beta, scale = 0.25, 32.0
    args = dict(clip_low=0.2, clip_high=0.3, kl="k3" if kl == "none" else kl, kl_beta=beta, reduce=reduce)
    x = x.detach().requires_grad_()
    # the gradient that the forward foresees, and another one
    out = PL.policy_loss(x, labels, mask, adv, old_logp=old, ref_logits=ref_logits, ref_logp=ref_logp, **args,
                         grad_scale=scale if reduce == "token" else 1.0)
    grad, = torch.autograd.grad(out.loss, x, torch.tensor(scale, device=DEV))
    xd = x.detach().double().requires_grad_()
    wide = lambda t: None if t is None else t.double()             # noqa: E731
    want = PL.policy_loss_ref(xd, labels, mask.double(), adv.double(), wide(old), wide(ref_logits), wide(ref_logp), **args)
    want_grad, = torch.autograd.grad(want.loss, xd, torch.tensor(scale, device=DEV, dtype=torch.float64))
    keep = mask != 0
    _near(out.logp, want.logp, keep * ROW + 2.0 ** -24 * want.logp.abs(), "logp")
    _near(out.clipped, want.clipped, 2.0 ** -22, "clipped")
    # each row: |r A| and the slope of the KL, times the error of its log-probability
    adv2 = (adv if adv.dim() == 2 else adv[:, None]).double().abs().expand(n, s)
    ratio = torch.ones_like(logp) if old is None else (logp - old.double()).exp()
    log_q = log_ratio = torch.zeros_like(p)
    if ref_logits is not None:
        log_q = ref_logits.double().log_softmax(-1)
        log_ratio = xd.detach().log_softmax(-1) - log_q
    rise = torch.zeros_like(logp)
    bend = torch.zeros_like(logp)                                  # slope of the slope
    if kl == "full":
        rise = (p * (log_ratio.abs() + 1)).sum(-1) + 1
    elif kl != "none":
        ref = log_q.gather(-1, labels[..., None])[..., 0] if ref_logits is not None else ref_logp.double()
        d = logp - ref
        rise = {"kl": torch.ones_like(d), "abs": torch.ones_like(d), "mse": d.abs(), "k3": torch.expm1(-d).abs()}[kl] + ROW
        bend = {"kl": 0 * d, "abs": 0 * d, "mse": torch.ones_like(d), "k3": (-d).exp()}[kl]
    off_row = 2 * ROW * (ratio * adv2 + beta * rise)               # policy and reference
    w = mask.double()
    share = w / w.sum()
    if reduce == "sequence":
        length = w.sum(-1, keepdim=True)
        weight = w / length.clamp(min=1e-30) / (length > 0).sum()
    else:
        weight = share
    _near(out.kl, want.kl, (2 * ROW * rise * share).sum() + 2.0 ** -24 * want.kl.abs(), "kl")
    _near(out.loss, want.loss.detach(), (off_row * weight).sum() + 2.0 ** -24 * want.loss.detach().abs(), "loss")
    slope = (ratio * adv2 + beta * (rise if kl != "full" else 0 * rise)) * weight * scale
    off_slope = (ratio * adv2 + beta * bend) * 2 * ROW * weight * scale + 2.0 ** -21 * slope
    hot = torch.zeros_like(p).scatter_(-1, labels[..., None], 1.0)
    bound = torch.finfo(dtype).eps / 2 * want_grad.abs() + (off_slope + 2.0 ** -20 * slope)[..., None] * (p + hot) \
        + 2 * ROW * slope[..., None] * p + _tiny(dtype)
    if kl == "full":                                               # b p ((log p - log q) - KL): p and the bracket
        pull = (beta * weight * scale)[..., None] * p
        bound = bound + pull * (2 * ROW * (log_ratio.abs() + want.kl.abs() + rise[..., None]) + 4 * ROW * rise[..., None])
    _near(grad, want_grad, bound, "gradient")
    assert not grad[~keep].any()


@pytest.mark.parametrize("kl", ["kl", "abs", "mse", "k3"])
@pytest.mark.parametrize("n,s,v,dtype,order,reduce", [
    (2, 6, 50257, torch.bfloat16, "bsv", "token"), (5, 5, 9001, torch.float32, "padded", "sequence"),
    (3, 6, 32001, torch.float16, "sbv", "token")])
def test_policy_loss_whose_reference_is_read_first(n, s, v, dtype, order, reduce, kl, monkeypatch):
    """As large batches have it: the reference's log-probabilities before the policy's one reading."""
    monkeypatch.setattr(PL, "_REF_FIRST", 0)
    test_policy_loss_matches_its_formula(n, s, v, dtype, order, kl, reduce)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("v", [40, 3000, 20001])
def test_loss_rows_of_extreme_logits(v, dtype):
    """Masked words of -inf and of the lowest number, labels on them, rows of nothing else, inf and NaN in kept and in masked
    rows, labels outside of the vocabulary: what the formula gives in 64 bits, and masked rows leave nothing at all."""
    n, s = 2, 12
    x, labels = _logits(n, s, v, dtype, seed=3)
    low = torch.finfo(dtype).min
    labels[:] = 5
    mask = torch.ones(n, s, device=DEV)
    x[0, 1, ::2] = -float("inf")
    x[0, 2, 1:4] = low
    x[0, 3, 10:] = low
    x[1, 0] = low                                                 # the row's lowest numbers are all there is
    x[1, 1, 5] = low
    x[1, 2, :5] = -float("inf")
    for j, bad in ((4, float("nan")), (5, float("inf")), (6, -float("inf"))):
        x[0, j] = bad
        mask[0, j] = 0
        labels[0, j] = -100
    ref = x.clone()
    ref[0, 7, 3] = -float("inf")
    x[0, 7, 3] = -float("inf")                                    # impossible for both: no part of the KL
    for full in (False, True):
        xl = x.detach().requires_grad_()
        adv = torch.linspace(-1, 1, n * s, device=DEV).view(n, s)
        kw = dict(ref_logits=ref, kl="full" if full else "kl", kl_beta=0.5)
        out = PL.policy_loss(xl, labels, mask, adv, **kw)
        grad, = torch.autograd.grad(out.loss, xl)
        xd = x.double().requires_grad_()
        want = PL.policy_loss_ref(xd, labels, mask.double(), adv.double(), ref_logits=ref.double(),
                                  **{k: t for k, t in kw.items() if k != "ref_logits"})
        want_grad, = torch.autograd.grad(want.loss, xd)
        # label 5 of row (1, 1) is at the lowest number: log-probabilities of that size are kept to their rounding
        _near(out.logp, want.logp, ROW + 2.0 ** -23 * want.logp.abs(), "logp")
        if not full:
            _near(out.kl, want.kl, 4 * ROW, "kl")                 # reference and policy are alike: the difference of two equal numbers
        ok = mask != 0
        weight = 1.0 / float(mask.sum())
        _near(grad[ok], want_grad[ok], torch.finfo(dtype).eps / 2 * want_grad[ok].abs() + 16 * ROW * weight + _tiny(dtype), "gradient")
        assert not grad[mask == 0].any() and bool(grad.isfinite().all())
    # kept rows that have no log-probability: NaN, and only in their own sequence
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[1, 3, 2] = bad
        out = PL.preference_loss(y, labels, mask, 0.1)
        assert out.logp[0].isfinite() and out.logp[1].isnan() and out.loss.isnan()
    y = x.clone()
    y[1, 3] = -float("inf")
    assert PL.preference_loss(y, labels, mask, 0.1).logp[1].isnan()
    for label in (-1, v):
        other = labels.clone()
        other[1, 3] = label
        out = PL.preference_loss(x, other, mask, 0.1)
        assert out.logp[0].isfinite() and out.logp[1].isnan()
        assert PL.policy_loss(x, other, mask, mask).logp[1, 3].isnan()
    y = x.clone()
    y[1, 3, 5] = -float("inf")                                    # a label of probability zero
    out = PL.preference_loss(y.requires_grad_(), labels, mask, 0.1)
    assert float(out.logp[1].detach()) == -float("inf") and float(out.loss.detach()) == 0.0
    grad, = torch.autograd.grad(out.loss, y)
    assert bool(grad.isfinite().all())
    out = PL.preference_loss(y.detach().flip(0), labels.flip(0), mask.flip(0), 0.1)
    assert float(out.loss) == float("inf")


def test_losses_of_batches_that_keep_nothing():
    x, labels = _logits(4, 6, 100, torch.bfloat16)
    x.requires_grad_()
    none = torch.zeros(4, 6, device=DEV)
    out = PL.preference_loss(x, labels, none, 0.1)
    assert abs(float(out.loss.detach()) - 0.6931471805599453) < 2.0 ** -23 and not out.logp.any()
    assert not torch.autograd.grad(out.loss, x)[0].any()
    for reduce in ("token", "sequence"):
        out = PL.policy_loss(x, labels, none, none, reduce=reduce)
        assert float(out.loss.detach()) == 0.0 and float(out.kl) == 0.0 and float(out.clipped) == 0.0
        assert not torch.autograd.grad(out.loss, x)[0].any()
    y, short = x.detach()[:, :0].requires_grad_(), labels[:, :0]
    out = PL.preference_loss(y, short, none[:, :0], 0.1)
    assert abs(float(out.loss.detach()) - 0.6931471805599453) < 2.0 ** -23
    assert torch.autograd.grad(out.loss, y)[0].shape == (4, 0, 100)
    assert float(PL.policy_loss(y, short, none[:, :0], none[:, :0]).loss.detach()) == 0.0


def test_policy_gradients_of_long_rows_that_are_not_kept_or_not_asked_for():
    x, labels = _logits(3, 50, 20000, torch.bfloat16)
    adv, mask = torch.ones(3, 50, device=DEV), torch.zeros(3, 50, device=DEV)
    x.requires_grad_()
    for kept in (0, 1, 2):                                         # rows that leave something: none, one, two of one sequence
        if kept:
            mask[1, 7 * kept] = 1.0
        for reduce in ("token", "sequence"):
            for scale in (1.0, 3.0, 0.0, float("nan")):
                out = PL.policy_loss(x, labels, mask, adv, reduce=reduce, grad_scale=scale)
                grad, = torch.autograd.grad(out.loss, x)
                assert not grad[mask == 0].any() and bool(grad.isfinite().all()) and bool(grad[mask != 0].any()) == bool(kept)
                want = PL.policy_loss_ref(x.detach().double().requires_grad_(), labels, mask.double(), adv.double(), reduce=reduce).loss
                _near(out.loss.detach(), want.detach(), 2.0 ** -22, "loss")
    # nobody asks for a gradient: none is written
    y = x.detach()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = PL.policy_loss(y, labels, mask, adv)
    assert not out.loss.requires_grad and torch.cuda.max_memory_allocated() - before < y.numel()


@pytest.mark.parametrize("op", ["preference", "policy", "foreseen", "not foreseen", "full", "router"])
def test_losses_repeat_bit_by_bit_on_any_stream_and_in_graphs(op):
    """The same inputs give the same bits: again, on another stream, with a second call in between, and replayed from a CUDA graph
    whose inputs have changed since it was captured."""
    n, s, v = 4, 130, 9000
    x, labels = _logits(n, s, v, torch.bfloat16)
    if op == "router":
        x = x.view(-1, 72)
    mask = _mask(n, s, 1)
    ref = x + 0.25
    x.requires_grad_()

    def once():
        if op == "preference":
            out = PL.preference_loss(x, labels, mask, 0.1, ref_logits=ref)
            outs = [out.loss, out.logp]
        elif op == "policy":
            outs = [PL.policy_loss(x, labels, mask, mask, ref_logits=ref, kl_beta=0.1).loss]
        elif op in ("foreseen", "not foreseen"):
            outs = [PL.policy_loss(x, labels, mask, mask, ref_logp=-mask, kl_beta=0.1, grad_scale=1.0 if op == "foreseen" else 2.0).loss]
        elif op == "full":
            outs = [PL.policy_loss(x, labels, mask, mask, ref_logits=ref, kl="full", kl_beta=0.1).loss]
        else:
            out = MO.balanced_router(x, 3)
            outs = [out.weights, out.balance, out.z]
        grad, = torch.autograd.grad(outs, [x], [torch.ones_like(o) for o in outs])
        return [o.detach().clone() for o in outs] + [grad]

    def same(a, b):
        return all(torch.equal(p, q) for p, q in zip(a, b))

    first = once()
    assert same(first, once())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            side = once()
    here = once()                                                  # at the same time as the other stream's
    torch.cuda.synchronize()
    assert same(first, side) and same(first, here)
    graphs, kept = [], []
    for _ in range(2):                                             # two graphs over the same inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append(once())
        graphs.append(graph)
    with torch.no_grad():
        x.mul_(0.5)
    want = once()
    assert not same(first, want)
    for graph in graphs + graphs[::-1]:
        graph.replay()
    torch.cuda.synchronize()
    assert same(want, kept[0]) and same(want, kept[1])


def test_loss_gradients_reach_what_asked_for_them():
    x, labels = _logits(2, 4, 50, torch.float32)
    mask = torch.ones(2, 4, device=DEV)
    x.requires_grad_()
    out = PL.preference_loss(x, labels, mask, 0.1)
    assert not out.ref_logp.requires_grad
    both, = torch.autograd.grad([out.loss, out.logp], x, [torch.tensor(2.0, device=DEV), torch.tensor([0.5, 0.0], device=DEV)], retain_graph=True)
    one, = torch.autograd.grad(out.loss, x, torch.tensor(2.0, device=DEV), retain_graph=True)
    two, = torch.autograd.grad(out.logp, x, torch.tensor([0.5, 0.0], device=DEV))
    # three gradients of one row: each is its coefficient, rounded once, times the same p
    _near(both, (one + two).double(), 2.0 ** -21 * (one.abs() + two.abs()).double(), "sum of both")
    out = PL.preference_loss(x, labels, mask, 0.1)
    again, = torch.autograd.grad(out.loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="a second time"):
        torch.autograd.grad(again.sum() + x.sum(), x)
    with torch.no_grad():
        assert torch.equal(PL.preference_loss(x, labels, mask, 0.1).loss, out.loss)
    out = PL.preference_loss(x, labels, mask, 0.1)
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.loss.backward()


@pytest.mark.parametrize("kl", ["k3", "k3 of tokens", "full"])
def test_a_policy_gradient_is_right_whatever_was_foreseen(kl):
    """The gradient for the foreseen gradient of the loss, for another one, and again through a retained graph; each a tensor of its
    own, and accumulated in ``.grad`` as it should be."""
    x, labels = _logits(2, 20, 9000, torch.float32)
    mask = _mask(2, 20, 2)
    ref = dict(ref_logp=-mask) if kl == "k3 of tokens" else dict(ref_logits=x + 0.3 * torch.randn_like(x))
    x.requires_grad_()
    loss = lambda scale: PL.policy_loss(x, labels, mask, mask, **ref, kl="full" if kl == "full" else "k3",     # noqa: E731
                                        kl_beta=0.2, grad_scale=scale).loss
    one = loss(1.0)
    first, = torch.autograd.grad(one, x, retain_graph=True)
    kept = first.clone()
    again, = torch.autograd.grad(one, x, retain_graph=True)
    twice, = torch.autograd.grad(one, x, torch.tensor(2.0, device=DEV))
    assert first.data_ptr() != again.data_ptr() and torch.equal(first, kept)
    # the same formula from statistics that were joined in another order: some roundings of numbers up to the coefficient
    top = kept.abs().max()
    _near(again, kept.double(), 2.0 ** -18 * top, "again")
    assert torch.equal(twice, 2 * again)                         # a power of two
    other, = torch.autograd.grad(loss(4.0), x)
    _near(other, kept.double(), 2.0 ** -18 * top, "not foreseen")
    scaled, = torch.autograd.grad(loss(4.0), x, torch.tensor(4.0, device=DEV))
    assert torch.equal(scaled, 4 * kept)
    for want in (1, 2):
        one = loss(1.0)
        one.backward(retain_graph=True)
        _near(x.grad, want * kept.double(), want * 2.0 ** -18 * top, "accumulated")
    one.backward()
    _near(x.grad, 3 * kept.double(), 3 * 2.0 ** -18 * top, "accumulated from a retained graph")


@pytest.mark.parametrize("full", [False, True])
def test_losses_over_a_split_vocabulary(full, monkeypatch):
    """Two tensor-parallel shares of the vocabulary, one after the other: what either share hands to the all-reduces is recorded
    and joined, and the third round, with the joined values, must give the loss and gradient of the whole vocabulary."""
    import torch.distributed as dist
    n, s, v, cut = 2, 9, 3000, 1500
    x, labels = _logits(n, s, v, torch.float32)
    mask = _mask(n, s, 5)
    x[0, 0, cut:] = -float("inf")
    ref = x + torch.randn_like(x) * 0.3
    adv = torch.randn(n, s, device=DEV)
    sent, rank_now = [[], []], [0]
    joined = []

    def all_reduce(t, op=None, group=None):
        i = len(sent[rank_now[0]])
        sent[rank_now[0]].append(t.clone())
        if i < len(joined):
            t.copy_(joined[i])

    def share(rank):
        rank_now[0] = rank
        sent[rank].clear()
        part = x[..., rank * cut:(rank + 1) * cut].detach().requires_grad_()
        ref_part = ref[..., rank * cut:(rank + 1) * cut]
        if full:
            loss = PL.policy_loss(part, labels, mask, adv, ref_logits=ref_part, kl="full", kl_beta=0.3).loss
        else:
            loss = PL.preference_loss(part, labels, mask, 0.2, ref_logits=ref_part).loss
        return loss.detach(), torch.autograd.grad(loss, part)[0]

    monkeypatch.setattr(PL, "_tensor_parallel", lambda: (2, rank_now[0], lambda: None))
    monkeypatch.setattr(dist, "all_reduce", all_reduce)
    share(0), share(1)
    joined.append(torch.maximum(sent[0][0], sent[1][0]))
    share(0), share(1)
    joined.append(sent[0][1] + sent[1][1])
    got = [share(0), share(1)]
    monkeypatch.undo()
    xl = x.detach().requires_grad_()
    if full:
        loss = PL.policy_loss(xl, labels, mask, adv, ref_logits=ref, kl="full", kl_beta=0.3).loss
    else:
        loss = PL.preference_loss(xl, labels, mask, 0.2, ref_logits=ref).loss
    grad, = torch.autograd.grad(loss, xl)
    coef = 0.2 if not full else 4.0                                # at most: beta, and |A| + |KL slope| over the kept tokens
    for r in (0, 1):
        _near(got[r][0], loss.detach(), 8 * ROW * s, "loss")
        _near(got[r][1], grad[..., r * cut:(r + 1) * cut], 8 * ROW * coef, "gradient")


# ---------------------------------------------------------------------------------------------- router
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,experts,k,masked,order", [
    (1, 2, 1, False, ""), (3, 1, 1, False, ""), (24, 8, 2, True, ""), (1000, 7, 3, True, "strided"), (777, 9, 8, False, "shifted"),
    (513, 16, 4, True, ""), (300, 33, 5, False, ""), (2000, 64, 6, True, "strided"), (257, 128, 8, False, ""), (90, 200, 2, True, ""),
    (65, 256, 1, False, "shifted"), (50, 300, 8, True, ""), (40, 512, 7, False, ""), (20000, 8, 1, True, ""), (0, 8, 2, False, "")])
def test_balanced_router_matches_its_formula(tokens, experts, k, masked, order, dtype):
    g = torch.Generator(device=DEV).manual_seed(tokens + experts)
    x = (torch.randn(tokens, experts, device=DEV, generator=g) * 2).to(dtype)
    if tokens > 2:
        x[1] = float(x[1, 0])                                          # all equal: the lowest indices
        x[2, ::2] = 0.0
        x[2, 1::2] = -0.0                                          # the same number
    if order == "strided":
        wide = torch.zeros(tokens, experts + 3, device=DEV, dtype=dtype)
        wide[:, :experts] = x
        x = wide[:, :experts]
    elif order == "shifted":
        x = torch.empty(x.numel() + 8, device=DEV, dtype=dtype)[3:3 + x.numel()].view_as(x).copy_(x)
    mask = torch.rand(tokens, device=DEV, generator=g) > 0.3 if masked else None
    x = x.detach().requires_grad_()
    out = MO.balanced_router(x, k, token_mask=mask)
    gw = torch.randn(tokens, k, device=DEV, generator=g)
    gb, gz = torch.tensor(0.7 * tokens, device=DEV), torch.tensor(0.01 * tokens, device=DEV)
    grad, = torch.autograd.grad([out.weights, out.balance, out.z], [x], [gw, gb, gz])
    xd = x.detach().double().requires_grad_()
    want = MO.balanced_router_ref(xd, k, mask)
    want_grad, = torch.autograd.grad([want.weights, want.balance, want.z], [xd], [gw.double(), gb.double(), gz.double()])
    assert torch.equal(out.experts, want.experts) and torch.equal(out.counts, want.counts)
    # a weight is a quotient of exponentials whose arguments are below 16 in size, or of one and their sum: 2^-19 relative
    _near(out.weights, want.weights.detach(), 2.0 ** -19 * want.weights.detach(), "weights")
    # column sums add up to 20000 / (blocks * groups) probabilities in a row, each off by 2^-19 of itself
    _near(out.balance, want.balance.detach(), 2.0 ** -18 * want.balance.detach(), "balance")
    _near(out.z, want.z.detach(), 2.0 ** -18 * (want.z.detach() + want.z.detach().sqrt()), "z")
    p = xd.detach().softmax(-1)
    kept = torch.ones(tokens, device=DEV, dtype=torch.float64) if mask is None else mask.double()
    count = kept.sum().clamp(min=1)
    load = torch.zeros(experts, device=DEV, dtype=torch.float64).index_add_(0, want.experts.reshape(-1), kept.repeat_interleave(k)) / (count * k)
    mass = p.gather(1, want.experts).sum(1, keepdim=True) if k > 1 else torch.ones(tokens, 1, device=DEV, dtype=torch.float64)
    # terms of dp: 2 |gw| / mass at the chosen experts, the balance term everywhere; their mean; the z term
    chosen = torch.zeros_like(p).scatter_(1, want.experts, (gw.double().abs() + (gw.double().abs() * want.weights.detach()).sum(1, keepdim=True)) / mass)
    size = chosen + (float(gb) * experts * load)[None] * kept[:, None] / count
    size = size + (size * p).sum(1, keepdim=True) + (2 * float(gz) * xd.detach().logsumexp(1).abs() * kept / count)[:, None]
    _near(grad, want_grad, torch.finfo(dtype).eps / 2 * want_grad.abs() + 2.0 ** -17 * p * size + _tiny(dtype), "gradient")


def test_balanced_router_of_extreme_logits():
    """NaN is above everything (as in a sort), infinities keep their order; a padded token with NaN leaves the losses alone."""
    x = torch.randn(6, 16, device=DEV).to(torch.bfloat16)
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3, 4:] = -float("inf")
    x[4] = torch.finfo(torch.bfloat16).min
    x[5, 7] = torch.finfo(torch.bfloat16).max
    keep = torch.tensor([True, False, False, True, True, True], device=DEV)
    out = MO.balanced_router(x, 4, token_mask=keep)
    want = MO.balanced_router_ref(x.double(), 4, keep)
    assert torch.equal(out.experts, want.experts) and int(out.experts[1, 0]) == 3 and int(out.experts[2, 0]) == 5
    ok = keep
    _near(out.weights[ok], want.weights[ok], 2.0 ** -19, "weights")
    assert bool(out.weights[1].isnan().all())
    _near(out.balance, want.balance, 2.0 ** -18 * want.balance, "balance")
    assert bool(torch.isfinite(out.balance))
    none = MO.balanced_router(x, 4, token_mask=torch.zeros_like(keep))
    assert float(none.balance) == 0.0 and float(none.z) == 0.0 and torch.equal(none.counts, out.counts)


# ---------------------------------------------------------------------------------------------- together, as they are used
def test_expert_model_trains_on_preferences_with_its_router_losses():
    """Router, experts and head, and on their logits the preference loss, a clipped policy loss, balance and z loss, as one objective:
    loss and all gradients against the same model of plain statements in 64 bits.  Everything is in 32 bits; products of up to 64
    terms, four in a row, stay within 2^-13 of the largest gradient."""
    torch.manual_seed(0)
    n, s, h, experts, v = 4, 33, 64, 8, 1003
    hidden = torch.randn(n * s, h, device=DEV)
    params = [torch.randn(experts, h, device=DEV) * 0.3, torch.randn(experts, h, h, device=DEV) / 8, torch.randn(v, h, device=DEV) / 8]
    labels, mask = torch.randint(0, v, (n, s), device=DEV), _mask(n, s, 3)
    old, adv = -torch.rand(n, s, device=DEV) - 6, torch.randn(n, device=DEV)
    tokens = mask.reshape(-1) != 0

    def objective(wr, we, wv, x, mask, old, adv, kernels):
        logits = x @ wr.t()
        route = MO.balanced_router(logits, 2, token_mask=tokens) if kernels else MO.balanced_router_ref(logits, 2, tokens)
        picked = torch.einsum("th,tkgh->tkg", x, we[route.experts]).tanh()
        out = (picked * route.weights.to(x.dtype)[..., None]).sum(1)
        words = (out @ wv.t()).view(n, s, v)
        prefer, policy = (PL.preference_loss, PL.policy_loss) if kernels else (PL.preference_loss_ref, PL.policy_loss_ref)
        a = prefer(words, labels, mask, 0.1)
        b = policy(words, labels, mask, adv, old_logp=old, ref_logits=words.detach() * 0.9, kl="full", kl_beta=0.1)
        return a.loss - 0.01 * a.logp.mean() + b.loss + 0.01 * route.balance + 1e-3 * route.z

    def run(dtype, kernels):
        w = [p.to(dtype).requires_grad_() for p in params]
        loss = objective(*w, *(t.to(dtype) for t in (hidden, mask, old, adv)), kernels)
        return [loss.detach()] + list(torch.autograd.grad(loss, w))
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        got, want = run(torch.float32, True), run(torch.float64, False)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = tf32
    for a, b in zip(got, want):
        _near(a, b, 2.0 ** -13 * b.abs().max(), "loss and gradients")


@pytest.mark.parametrize("kind", ["dpo", "clipped", "moe"])
def test_post_training_steps_on_a_gpu(kind):
    import os
    import subprocess
    import sys
    from common import ROOT, free_port
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT=str(free_port()), WORLD_SIZE="1", RANK="0", LOCAL_RANK="0")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "workers", "post_training_worker.py"), kind], env=env,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "POST_TRAINING_OK" in r.stdout, (r.stdout + r.stderr)[-4000:]


@pytest.mark.parametrize("dtype,v", [(torch.bfloat16, 9001), (torch.float32, 2051)])
def test_gradients_of_sliced_logits_lie_as_the_logits_do(dtype, v):
    """Logits without their last position, of an odd vocabulary: the gradient's rows begin where the logits' do, what lies between them
    is not touched, and the whole gradient is the sliced one with zeros behind."""
    whole, labels = _logits(3, 8, v, dtype)
    whole.requires_grad_()
    mask = torch.ones(3, 7, device=DEV)
    for scale in (1.0, 2.0):                                       # foreseen and not
        for op in ("policy", "preference"):
            x = (whole if op == "policy" else whole[:2])[:, :-1]
            n = x.shape[0]
            if op == "policy":
                loss = PL.policy_loss(x, labels[:, :-1], mask, mask, grad_scale=scale).loss
            else:
                loss = PL.preference_loss(x, labels[:2, :-1], mask[:2], 0.1).loss
            part, all_of_it = torch.autograd.grad(loss, [x, whole])
            assert part.stride() == x.stride() and part.data_ptr() % 16 == x.data_ptr() % 16
            assert torch.equal(all_of_it[:n, :-1], part) and not all_of_it[:, -1].any() and not all_of_it[n:].any()
    # logits that lie too far apart for that, or on one another
    apart = whole.detach()[:, ::4].requires_grad_()
    loss = PL.policy_loss(apart, labels[:, ::4], mask[:, :2], mask[:, :2]).loss
    assert torch.autograd.grad(loss, apart)[0].is_contiguous()
    same = whole.detach()[:1].expand(4, 8, v).requires_grad_()
    loss = PL.policy_loss(same, labels[:1].expand(4, 8), mask[:1, :1].expand(4, 8), mask[:1, :1].expand(4, 8)).loss
    grad, = torch.autograd.grad(loss, same)
    assert grad.is_contiguous() and torch.equal(grad[0], grad[3])


@pytest.mark.parametrize("op", ["preference", "policy", "not foreseen", "full"])
def test_losses_of_more_logits_than_32_bits_number(op):
    """More than 2^31 logits of which the last positions of two sequences are kept: loss and gradient are those of these positions
    alone, and zero elsewhere.  Both sides round a gradient once to bf16, from coefficients and probabilities that are ROW apart."""
    n, s, v, last = 44, 1000, 50304, 3
    pair = [n // 2 - 1, n - 1]
    x = torch.empty(n, s, v, device=DEV, dtype=torch.bfloat16).normal_()
    y = torch.empty_like(x).normal_() if op == "full" else None
    labels = torch.randint(0, v, (n, s), device=DEV)
    mask = torch.zeros(n, s, device=DEV)
    mask[pair, -last:] = 1.0

    def run(x, labels, mask, y):
        x = x.detach().requires_grad_()
        if op == "preference":
            out = PL.preference_loss(x, labels, mask, 0.5)
            grad, = torch.autograd.grad(out.loss, x, torch.tensor(float(x.shape[0] // 2), device=DEV))
            return out.logp[-1].detach(), grad
        out = PL.policy_loss(x, labels, mask, mask, ref_logits=y, kl="full" if op == "full" else "k3", kl_beta=0.3,
                             grad_scale=2.0 if op == "not foreseen" else 1.0)
        return out.loss.detach(), torch.autograd.grad(out.loss, x)[0]

    got, grad = run(x, labels, mask, y)
    few = [t[pair][:, -last:].clone() if t is not None else None for t in (x, labels, mask, y)]
    want, want_grad = run(*few)
    _near(got, want.double(), 8 * ROW * (1 + want.double().abs()), "value")
    eps = torch.finfo(torch.bfloat16).eps
    size = want_grad.double().abs()
    # a probability is below 2^-8 here, a coefficient at most twice the largest gradient, which stands at a label
    _near(grad[pair][:, -last:], want_grad.double(), eps * size + 8 * ROW * size.max() * (2.0 ** -8 + (size > size.max() / 8)), "gradient")
    grad[pair, -last:] = 0
    assert not grad.any()


def test_router_of_more_logits_than_32_bits_number():
    tokens, experts, k, last = 4_300_000, 512, 4, 999
    x = torch.empty(tokens, experts, device=DEV, dtype=torch.bfloat16).normal_().requires_grad_()
    out = MO.balanced_router(x, k)
    few = x.detach()[-last:].clone().requires_grad_()
    want = MO.balanced_router(few, k)
    assert torch.equal(out.experts[-last:], want.experts) and torch.equal(out.weights[-last:], want.weights)
    assert int(out.counts.sum()) == tokens * k
    g = torch.zeros(tokens, k, device=DEV)
    g[-last:] = torch.randn(last, k, device=DEV)
    grad, = torch.autograd.grad(out.weights, x, g)
    want_grad, = torch.autograd.grad(want.weights, few, g[-last:].contiguous())
    assert torch.equal(grad[-last:], want_grad) and not grad[:-last].any()
