"""Preference and policy loss on a GPU where their digits, their graphs and their choice of a path could differ from what is documented.

ROW bounds what a row's log-probability is off by (``test_policy_losses_gpu.py`` derives it); where a log-probability is exact by
construction the tests below allow roundings of the result alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from gpt_neox_b200.ops import policy_losses as PL

DEV = "cuda"
ROW = 2.0 ** -18


def test_pairs_are_joined_in_64_bits():
    """A vocabulary of two words 1024 apart has the log-probabilities 0 and -1024 exactly, so z is exact in 64 bits.  What is left is
    one rounding of the loss (2^-24 of it) and, in the gradient, the roundings of the pair's coefficient, of its product with the
    gradient of the loss, and of the result."""
    x = torch.zeros(2, 1, 2, device=DEV)
    x[0, 0, 1] = -1024.0
    x[1, 0, 0] = -1024.0
    mask = torch.ones(2, 1, device=DEV)
    for label, sign in ((0, 1.0), (1, -1.0)):                      # the chosen answer more probable, and less
        labels = torch.full((2, 1), label, device=DEV)
        for size in (1e-3, 0.1, 0.7, 2.3, 5.1, 9.7, 13.3, 17.9, 25.1, 33.7, 51.3, 71.9):
            for eps in (0.0, 0.1):
                xl = x.clone().requires_grad_()
                out = PL.preference_loss(xl, labels, mask, size / 1024.0, label_smoothing=eps)
                grad, = torch.autograd.grad(out.loss, xl)
                z = torch.tensor(sign * (size / 1024.0 * 1024.0), dtype=torch.float64)
                want = -(1 - eps) * torch.nn.functional.logsigmoid(z) - eps * torch.nn.functional.logsigmoid(-z)
                assert abs(float(out.loss.detach().double() - want)) <= 2.0 ** -24 * float(want) * 1.001, (size, sign, eps)
                slope = -size / 1024.0 * ((1 - eps) * torch.sigmoid(-z) - eps * torch.sigmoid(z))
                hot = abs(float(grad[0, 0, 1].double()))          # coefficient * (1 - 0) or (0 - 1), whichever word is impossible
                assert abs(hot - (abs(float(slope)) if label else 0.0)) <= 2.0 ** -22 * abs(float(slope)), (size, sign, eps)


def test_reference_read_first_keeps_the_digits_of_improbable_labels(monkeypatch):
    """Labels of log-probabilities near -3000: their difference between policy and reference is as near as below the size from which
    the reference is read first, whose log-probabilities in 32 bits would be off by up to 2^-13."""
    n, s, v = 1, 16, 9000
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(n, s, v, device=DEV, generator=g) * 2
    y = x + 0.3 * torch.randn(n, s, v, device=DEV, generator=g)
    labels = torch.randint(0, v, (n, s), device=DEV, generator=g)
    x.scatter_(2, labels[..., None], -3000.0)
    y.scatter_(2, labels[..., None], -3000.25)
    lp = lambda t: t.double().log_softmax(-1).gather(-1, labels[..., None])[..., 0]       # noqa: E731
    want = lp(x) - lp(y)
    for first in (0, 1 << 62):
        monkeypatch.setattr(PL, "_REF_FIRST", first)
        for j in range(s):
            mask = torch.zeros(n, s, device=DEV)
            mask[0, j] = 1.0
            out = PL.policy_loss(x.requires_grad_(), labels, mask, mask, ref_logits=y, kl="kl", kl_beta=0.1)
            assert abs(float(out.kl.double() - want[0, j])) <= 2 * ROW + 2.0 ** -24 * abs(float(want[0, j])), (first, j)


@pytest.mark.parametrize("kl", ["kl", "abs", "mse", "k3"])
@pytest.mark.parametrize("order", ["bsv", "sbv"])
def test_reference_equal_to_the_policy_pulls_nowhere(kl, order, monkeypatch):
    """As at the first step of training, whatever the batch's size: d is zero, and with it the slope of |d|, which is none or the whole
    weight.  The other slopes follow d, which is off by 2 ROW at most."""
    n, s, v = 3, 40, 9000
    g = torch.Generator(device=DEV).manual_seed(1)
    x = (torch.randn(*((n, s) if order == "bsv" else (s, n)), v, device=DEV, generator=g) * 2).to(torch.bfloat16)
    x = x if order == "bsv" else x.transpose(0, 1)
    labels = torch.randint(0, v, (n, s), device=DEV, generator=g)
    mask = torch.ones(n, s, device=DEV)
    for first in (0, 1 << 62):
        monkeypatch.setattr(PL, "_REF_FIRST", first)
        xl = x.detach().requires_grad_()
        out = PL.policy_loss(xl, labels, mask, 0 * mask, ref_logits=x.clone(), kl=kl, kl_beta=1.0)
        grad, = torch.autograd.grad(out.loss, xl)
        assert abs(float(out.kl)) <= 2 * ROW
        if kl == "kl":
            assert float(grad.abs().max()) > 0.9 / (n * s)         # its slope is one everywhere
        else:
            assert float(grad.abs().max()) <= (0.0 if kl == "abs" else 2 * ROW / (n * s)), (first, float(grad.abs().max()))


def test_clipped_tokens_leave_nothing_whatever_gradient_was_foreseen():
    """A slope of zero gives zeros, also where the gradient of the loss is infinite and was foreseen."""
    x = torch.randn(2, 6, 9000, device=DEV)
    labels = torch.zeros(2, 6, dtype=torch.long, device=DEV)
    mask, adv = torch.ones(2, 6, device=DEV), torch.ones(2, 6, device=DEV)
    old = x.log_softmax(-1)[..., 0] - 1.0                          # a ratio of e: clipped, since the advantage is positive
    old[0, 0] += 1.0                                              # but for one token
    for foreseen in (float("inf"), 1.0):
        xl = x.clone().requires_grad_()
        out = PL.policy_loss(xl, labels, mask, adv, old_logp=old, grad_scale=foreseen)
        grad, = torch.autograd.grad(out.loss, xl, torch.tensor(float("inf"), device=DEV))
        rest = grad.flatten(0, 1)[1:]
        assert not rest.any() and not bool(rest.isnan().any()), foreseen
        assert not bool(grad[0, 0].isfinite().any()), foreseen


def test_a_captured_backward_of_an_eager_forward_writes_its_gradient_at_every_replay():
    """The foreseen gradient is written once, by the forward: a backward that is replayed without it computes its own each time, and
    the eager backward after it still finds the right one."""
    x = torch.randn(2, 20, 9000, device=DEV)
    labels = torch.randint(0, 9000, (2, 20), device=DEV)
    mask = torch.ones(2, 20, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        leaf = x.clone().requires_grad_()
        y = leaf * 1.0                                            # what is asked for is not a leaf
        one = torch.ones((), device=DEV)
        warm, = torch.autograd.grad(PL.policy_loss(y, labels, mask, mask).loss, y, one)
        want = warm.clone()
        loss = PL.policy_loss(y, labels, mask, mask).loss
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        grad, = torch.autograd.grad(loss, y, one, retain_graph=True)
        grad.mul_(0.5)                                            # as a clipping of gradients does
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    # the same formula from the same statistics: roundings of the coefficient's products
    top = want.abs().max()
    assert float((grad - 0.5 * want).abs().max()) <= 2.0 ** -18 * float(top)
    with torch.cuda.stream(stream):
        again, = torch.autograd.grad(loss, y, one)
    torch.cuda.synchronize()
    assert float((again - want).abs().max()) <= 2.0 ** -18 * float(top)


def test_an_eager_backward_of_a_captured_forward_has_a_gradient_of_its_own():
    """The forward is replayed, its backward is not part of the graph: a gradient that was handed out stays as it is when the forward
    is replayed on other logits."""
    x = torch.randn(2, 20, 9000, device=DEV)
    labels = torch.randint(0, 9000, (2, 20), device=DEV)
    mask = torch.ones(2, 20, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        base = x.clone()
        leaf = base.requires_grad_()
        one = torch.ones((), device=DEV)
        torch.autograd.grad(PL.policy_loss(leaf * 1.0, labels, mask, mask).loss, leaf, one)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = leaf * 1.0
        loss = PL.policy_loss(y, labels, mask, mask).loss
    with torch.cuda.stream(stream):
        graph.replay()
        first, = torch.autograd.grad(loss, y, one, retain_graph=True)
        kept = first.clone()
        with torch.no_grad():
            base.mul_(0.25)
        graph.replay()
        second, = torch.autograd.grad(loss, y, one, retain_graph=True)
    torch.cuda.synchronize()
    assert torch.equal(first, kept)
    yl = (0.25 * x).requires_grad_()
    want, = torch.autograd.grad(PL.policy_loss(yl, labels, mask, mask).loss, yl, one)
    assert float((second - want).abs().max()) <= 2.0 ** -18 * float(want.abs().max())
    assert not torch.equal(first, second)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kl,ref", [("k3", "logits"), ("mse", "logits"), ("k3", "logp"), ("kl", "none")])
def test_clipped_loss_over_a_split_vocabulary(kl, ref, dtype, monkeypatch):
    """Two tensor-parallel shares of the vocabulary, one after the other: what either hands to the all-reduces is recorded and joined,
    and the third round, with the joined values, gives the loss and gradient of the whole vocabulary.  Either side's rows are off by
    ROW, their gradients rounded once."""
    import torch.distributed as dist
    n, s, v, cut = 3, 17, 6000, 3000
    g = torch.Generator(device=DEV).manual_seed(3)
    x = (torch.randn(n, s, v, device=DEV, generator=g) * 2).to(dtype)
    labels = torch.randint(0, v, (n, s), device=DEV, generator=g)
    labels[0, 0], labels[0, 1], labels[0, 2], labels[0, 3] = 0, cut - 1, cut, v - 1
    mask = (torch.rand(n, s, device=DEV, generator=g) > 0.4).float()
    mask[0, :4] = 1.0
    adv = torch.randn(n, s, device=DEV, generator=g)
    y = x + (0.3 * torch.randn(n, s, v, device=DEV, generator=g)).to(dtype)
    logp = x.double().log_softmax(-1).gather(-1, labels[..., None])[..., 0]
    old = (logp + 0.1 * torch.randn(n, s, device=DEV, generator=g)).float()
    stored = (logp + 0.2 * torch.randn(n, s, device=DEV, generator=g)).float()
    beta, sent, rank_now, joined = 0.3, [[], []], [0], []

    def all_reduce(t, op=None, group=None):
        i = len(sent[rank_now[0]])
        sent[rank_now[0]].append(t.clone())
        if i < len(joined):
            t.copy_(joined[i])

    def loss_of(x, y):
        x = x.detach().requires_grad_()
        given = {"logits": {"ref_logits": y}, "logp": {"ref_logp": stored}, "none": {}}[ref]
        out = PL.policy_loss(x, labels, mask, adv, old_logp=old, kl=kl, kl_beta=beta, reduce="sequence", **given)
        return out.loss.detach(), out.logp, out.kl, torch.autograd.grad(out.loss, x)[0]

    def share(rank):
        rank_now[0] = rank
        sent[rank].clear()
        at = slice(rank * cut, (rank + 1) * cut)
        return loss_of(x[..., at], y[..., at])

    with monkeypatch.context() as m:
        m.setattr(PL, "_tensor_parallel", lambda: (2, rank_now[0], lambda: None))
        m.setattr(dist, "all_reduce", all_reduce)
        share(0), share(1)
        joined.append(torch.maximum(sent[0][0], sent[1][0]))
        share(0), share(1)
        joined.append(sent[0][1] + sent[1][1])
        got = [share(0), share(1)]
    loss, lp, mean_kl, grad = loss_of(x, y)
    d = logp - (y.double().log_softmax(-1).gather(-1, labels[..., None])[..., 0] if ref == "logits" else stored.double())
    steep = {"k3": torch.exp(-d) + 1, "mse": d.abs() + 1, "kl": torch.ones_like(d)}[kl]      # of the estimate and of its slope
    ratio = (logp - old.double()).exp()
    most = float(((ratio * adv.double().abs() + beta * steep) * (mask != 0)).max())
    for r in (0, 1):
        assert abs(float(got[r][0] - loss)) <= 4 * ROW * most
        assert float((got[r][1] - lp).abs().max()) <= 4 * ROW and abs(float(got[r][2] - mean_kl)) <= 4 * ROW * float(steep.max())
        want = grad[..., r * cut:(r + 1) * cut].double()
        off = (got[r][3].double() - want).abs()
        assert bool((off <= torch.finfo(dtype).eps * want.abs() + 8 * ROW * most / n).all())


@pytest.mark.parametrize("dtype,v,spread,train", [(torch.bfloat16, 50304, 2.0, True), (torch.float32, 50432, 2.0, False),
                                                  (torch.float32, 9001, 2.0, True), (torch.bfloat16, 32000, 5.0, False)])
def test_log_probabilities_are_not_off_on_average(dtype, v, spread, train):
    """Half of the rows' log-probabilities, taken as the difference to their 64-bit values rounded to 32, within 3e-8: a loss of terms of
    either sign keeps its digits.  The lanes' roundings average out over a row (2^-22 each, over hundreds of lanes: 5e-9 and less).  What
    is left is the mean error of the exponential, from -5e-8 (of ex2) up by 1.3e-8 for every unit of the argument (log2 e in 32 bits):
    the words that count lie 2 to 6 below their lane's largest, and the factors of whole sums are corrected."""
    s = 96
    g = torch.Generator(device=DEV).manual_seed(v)
    x = torch.randn(1, s, v, device=DEV, generator=g, dtype=dtype).mul_(spread)
    labels = torch.randint(0, v, (1, s), device=DEV, generator=g)
    want = x.double().log_softmax(-1).gather(-1, labels[..., None])[..., 0]
    near = want.float()
    x.requires_grad_(train)
    off = []
    for j in range(s):
        mask = torch.zeros(1, s, device=DEV)
        mask[0, j] = 1.0
        off.append(PL.policy_loss(x, labels, mask, mask, ref_logp=near, kl="kl", kl_beta=0.1).kl.double() - (want - near.double())[0, j])
    off = torch.stack(off).abs()
    assert float(off.median()) <= 3e-8 and float(off.max()) <= ROW
