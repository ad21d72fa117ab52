"""The losses of post-training and of expert routing whose speed counts: a preference loss over pairs of sequences, a clipped
policy loss with a KL term, and the router of a mixture of experts with its balance and z losses.

A pass of a training case is the forward and the backward of one operator, as it stands between a model's logits and their
gradient; a pass of an evaluation case is the forward alone.  ``own`` chooses between this repository's operators and the same
mathematics in elementary torch operations.

Logits look like a language model's: a spread of a few units and a label that stands out.  Prompts and padding are masked, so a
part of the rows counts.  Which rows these are follows from the case alone, the values from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_KL = ("kl", "abs", "mse", "k3", "full")


def _loss_case(name, op, **over):
    """``n`` sequences of ``s`` tokens over ``vocab`` words; ``prompt``: the share of a sequence its prompt takes on average;
    ``ref``: what the reference model gives (none | logp | logits); ``order``: memory order of the logits, batch (``bsv``) or
    time (``sbv``) first; ``scale``: the loss scale the backward starts from; ``train`` off: no gradient is taken."""
    c = {"name": name, "op": op, "dtype": "bf16", "n": 2, "s": 128, "vocab": 50304, "prompt": 0.4, "padding": 0.2,
         "empty": False, "ref": "logp", "order": "bsv", "scale": 1.0, "train": True}
    c.update({"beta": 0.1, "smoothing": 0.0, "nll": 0.0} if op == "preference" else
             {"kl": "k3", "kl_beta": 0.05, "low": 0.2, "high": 0.2, "old": True, "reduce": "token", "adv": "token"})
    c.update(over)
    return c


def _router_case(name, **over):
    c = {"name": name, "op": "router", "dtype": "bf16", "tokens": 8192, "experts": 8, "k": 2, "padding": 0.0, "train": True,
         "scale": 1.0}
    c.update(over)
    return c


def listed():
    return [
        # One short pair with stored reference log-probabilities: the smallest preference step.
        _loss_case("dpo_one_pair", "preference", n=2, s=48, vocab=32000),
        # A micro-batch of four pairs over the vocabulary of the GPT configurations, the reference model beside the policy.
        _loss_case("dpo_pairs", "preference", n=8, s=1024, ref="logits"),
        # post-training/configs/llama3-8b-dpo.yml: two pairs of 8192 tokens, a tensor-parallel quarter of its vocabulary.
        _loss_case("dpo_long_shard", "preference", n=4, s=8192, vocab=32064, beta=0.01, prompt=0.3),
        # An unpadded vocabulary, time-first logits, fp16 with loss scaling, smoothed labels, a likelihood term on the chosen
        # answers and a pair that lost all its tokens to truncation.
        _loss_case("dpo_odd", "preference", dtype="fp16", n=6, s=333, vocab=50257, order="sbv", scale=1024.0, smoothing=0.1,
                   nll=0.2, ref="logits", empty=True),
        # Validation in single precision: no gradient.
        _loss_case("dpo_eval", "preference", dtype="fp32", n=4, s=512, vocab=50432, ref="logits", train=False),
        # One short completion: the smallest policy step.
        _loss_case("policy_one", "policy", n=1, s=37),
        # Online training on sampled completions with the sampler's log-probabilities and a stored reference.
        _loss_case("policy_tokens", "policy", n=8, s=1024),
        # The KL over the whole vocabulary against a reference model, averaged by sequence.
        _loss_case("policy_full", "policy", n=8, s=2048, vocab=50432, ref="logits", kl="full", reduce="sequence", adv="sequence"),
        # Odd sizes in fp16 with an unsymmetric clip and the squared-difference KL from reference logits.
        _loss_case("policy_odd", "policy", dtype="fp16", n=3, s=701, vocab=32001, ref="logits", kl="mse", scale=512.0, high=0.28),
        # configs/125M-moe.yml: eight sequences of 2048 tokens, eight experts, top-1, fp16 with loss scaling.
        _router_case("router_8", dtype="fp16", tokens=16384, k=1, scale=256.0),
        # Many experts, several of them a token, padded sequences.
        _router_case("router_128", tokens=32768, experts=128, k=8, padding=0.15),
        # A handful of tokens: the launch is what is paid for.
        _router_case("router_few", tokens=24, experts=64, k=4),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["preference", "preference", "policy", "policy", "router"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        scale = 2.0 ** rng.randint(6, 12) if dtype == "fp16" else 1.0
        train = rng.random() < 0.8
        if op == "router":
            experts = rng.choice([4, 8, 16, 64, 128, 256, rng.randint(2, 512)])
            c = _router_case("", dtype=dtype, scale=scale, train=train, tokens=_log_uniform(rng, 1, 65536), experts=experts,
                             k=min(experts, rng.randint(1, 8)), padding=rng.choice([0.0, rng.uniform(0.0, 0.5)]))
        else:
            more = {"dtype": dtype, "scale": scale, "train": train, "s": _log_uniform(rng, 1, 8192),
                    "vocab": rng.choice([32000, 50257, 50304, 50432, _log_uniform(rng, 500, 128256)]),
                    "prompt": rng.uniform(0.0, 0.8), "padding": rng.uniform(0.0, 0.5), "empty": rng.random() < 0.2,
                    "order": rng.choice(["bsv", "bsv", "sbv"])}
            if op == "preference":
                c = _loss_case("", op, **more, n=2 * _log_uniform(rng, 1, 16), ref=rng.choice(["none", "logp", "logits"]),
                               beta=rng.uniform(0.01, 0.5), smoothing=rng.choice([0.0, rng.uniform(0.0, 0.4)]),
                               nll=rng.choice([0.0, rng.uniform(0.0, 1.0)]))
            else:
                kl = rng.choice(_KL)
                c = _loss_case("", op, **more, n=_log_uniform(rng, 1, 32), kl=kl,
                               ref="logits" if kl == "full" else rng.choice(["none", "logp", "logits"]),
                               kl_beta=rng.uniform(0.01, 0.5), low=rng.uniform(0.1, 0.3), high=rng.uniform(0.1, 0.4),
                               old=rng.random() < 0.8, reduce=rng.choice(["token", "sequence"]),
                               adv=rng.choice(["token", "sequence"]))
        del c["name"]
        if work(c)["bytes"] <= limit:
            return c


# ---------------------------------------------------------------------------------------------- inputs
def _spans(c):
    """First and last kept position of every sequence: prompts and lengths that vary evenly around the case's shares."""
    n, s = c["n"], c["s"]
    first = [min(s - 1, int(c["prompt"] * s * (0.5 + (0.618034 * i) % 1.0))) for i in range(n)]
    last = [max(f + 1, s - int(c["padding"] * s * ((0.754878 * i) % 1.0))) for i, f in enumerate(first)]
    if c["empty"] and n > 1:
        first[-1] = last[-1] = 0
    return first, last


def _kept_rows(c):
    return sum(b - a for a, b in zip(*_spans(c)))


def _kept_tokens(c):
    return max(1, c["tokens"] - int(c["padding"] * c["tokens"]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "router":
        t, e, k = case["tokens"], case["experts"], case["k"]
        # some experts are liked more than others, as before a balance loss has worked
        logits = (torch.randn(t, e, device="cuda", generator=g) * 1.5 + torch.randn(e, device="cuda", generator=g)).to(dt)
        mask = None
        if case["padding"]:
            mask = torch.arange(t, device="cuda") < _kept_tokens(case)
        return {"case": case, "logits": logits.requires_grad_(case["train"]), "mask": mask,
                "dw": torch.randn(t, k, device="cuda", generator=g) * case["scale"],
                "dloss": torch.tensor(0.1 * t * case["scale"], device="cuda"),
                "dz": torch.tensor(1e-3 * t * case["scale"], device="cuda")}
    n, s, v = case["n"], case["s"], case["vocab"]
    shape = (n, s) if case["order"] == "bsv" else (s, n)
    logits = torch.randn(*shape, v, device="cuda", generator=g, dtype=dt).mul_(2.0)
    labels = torch.randint(0, v, shape, device="cuda", generator=g)
    logits.scatter_add_(2, labels[..., None], torch.full((*shape, 1), 9.0, device="cuda", dtype=dt))
    ref = None
    if case["ref"] == "logits":
        ref = torch.randn(*shape, v, device="cuda", generator=g, dtype=dt).mul_(0.3).add_(logits)
    if case["order"] == "sbv":
        logits, labels = logits.transpose(0, 1), labels.t().contiguous()
        ref = None if ref is None else ref.transpose(0, 1)
    first, last = (torch.tensor(x, device="cuda")[:, None] for x in _spans(case))
    at = torch.arange(s, device="cuda")[None]
    st = {"case": case, "labels": labels, "mask": ((at >= first) & (at < last)).float(), "ref_logits": ref, "ref_logp": None,
          "logits": logits.requires_grad_(case["train"]), "scale": torch.tensor(case["scale"], device="cuda")}
    noise = lambda *size: torch.randn(*size, device="cuda", generator=g)  # noqa: E731
    # what samplers and reference runs store beside the tokens
    logp = _token_logp(logits.detach(), labels).float() if case["ref"] == "logp" or case.get("old") else None
    if case["ref"] == "logp":
        st["ref_logp"] = logp + 0.1 * noise(n, s)
    if case["op"] == "preference":
        st["dlogp"] = torch.full((n,), -case["nll"] / n * case["scale"], device="cuda")
        st["dlogp"][n // 2:] = 0.0
    else:
        st["old_logp"] = logp + 0.15 * noise(n, s) if case["old"] else None
        st["advantages"] = noise(n, s) if case["adv"] == "token" else noise(n)
    return st


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    c = state["case"]
    if c["op"] == "preference":
        return _preference_own(state, c) if own else _preference_plain(state, c)
    if c["op"] == "policy":
        return _policy_own(state, c) if own else _policy_plain(state, c)
    return _router_own(state, c) if own else _router_plain(state, c)


def _preference_own(st, c):
    from gpt_neox_b200.ops.policy_losses import preference_loss
    out = preference_loss(st["logits"], st["labels"], st["mask"], beta=c["beta"], ref_logits=st["ref_logits"],
                          ref_logp=st["ref_logp"], label_smoothing=c["smoothing"])
    got = {"loss": out.loss.detach(), "logp": out.logp.detach(), "ref_logp": out.ref_logp}
    if c["train"]:
        got["grad"], = torch.autograd.grad([out.loss, out.logp], [st["logits"]], [st["scale"], st["dlogp"]])
    return got


def _policy_own(st, c):
    from gpt_neox_b200.ops.policy_losses import policy_loss
    out = policy_loss(st["logits"], st["labels"], st["mask"], st["advantages"], old_logp=st["old_logp"],
                      ref_logits=st["ref_logits"], ref_logp=st["ref_logp"], clip_low=c["low"], clip_high=c["high"], kl=c["kl"],
                      kl_beta=c["kl_beta"], reduce=c["reduce"])
    got = {"loss": out.loss.detach(), "logp": out.logp, "kl": out.kl, "clipped": out.clipped}
    if c["train"]:
        got["grad"], = torch.autograd.grad(out.loss, st["logits"], st["scale"])
    return got


def _router_own(st, c):
    from gpt_neox_b200.ops.moe_ops import balanced_router
    out = balanced_router(st["logits"], c["k"], token_mask=st["mask"])
    got = {"weights": out.weights.detach(), "experts": out.experts, "counts": out.counts, "balance": out.balance.detach(),
           "z": out.z.detach()}
    if c["train"]:
        got["grad"], = torch.autograd.grad([out.weights, out.balance, out.z], [st["logits"]], [st["dw"], st["dloss"], st["dz"]])
    return got


# ---------------------------------------------------------------------------------------------- plain forms
def _softmax_parts(x):
    """``exp(x - max)`` and its sum, in 32 bits, and the logarithm of the sum over the exponentials in 64."""
    xf = x.float()
    top = xf.amax(-1, keepdim=True)
    e = (xf - top).exp_()
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    return e, total, (top.double() + total.log())[..., 0]


def _token_logp(x, labels):
    """Log-probability of every label, in 64 bits from the sum on: a sequence adds thousands of them and a pair takes the
    difference of two such sums."""
    _, _, lse = _softmax_parts(x)
    return x.gather(-1, labels[..., None])[..., 0].double() - lse


def _logits_grad(e, total, labels, coef, dtype):
    """``coef * (onehot(label) - softmax)``."""
    p = e.mul_((-coef / total[..., 0]).float()[..., None])
    p.scatter_add_(-1, labels[..., None], coef.float()[..., None])
    return p.to(dtype)


def _preference_plain(st, c):
    x, labels, mask = st["logits"].detach(), st["labels"], st["mask"].double()
    e, total, lse = _softmax_parts(x)
    logp = ((x.gather(-1, labels[..., None])[..., 0].double() - lse) * mask).sum(-1)
    ref = torch.zeros_like(logp)
    if st["ref_logits"] is not None:
        ref = (_token_logp(st["ref_logits"], labels) * mask).sum(-1)
    elif st["ref_logp"] is not None:
        ref = (st["ref_logp"].double() * mask).sum(-1)
    half, eps = c["n"] // 2, c["smoothing"]
    z = c["beta"] * ((logp[:half] - logp[half:]) - (ref[:half] - ref[half:]))
    softplus = z.abs().neg().exp().log1p()
    loss = ((1 - eps) * (softplus + (-z).clamp(min=0)) + eps * (softplus + z.clamp(min=0))).mean()
    got = {"loss": loss.float(), "logp": logp.float(), "ref_logp": ref.float()}
    if c["train"]:
        right = 1 / (1 + (-z).exp())
        d = -c["beta"] / half * ((1 - eps) * (1 - right) - eps * right)
        coef = torch.cat([d, -d]) * st["scale"].double() + st["dlogp"].double()
        got["grad"] = _logits_grad(e, total, labels, coef[:, None] * mask, x.dtype)
    return got


def _policy_plain(st, c):
    x, labels, mask = st["logits"].detach(), st["labels"], st["mask"].double()
    e, total, lse = _softmax_parts(x)
    logp = x.gather(-1, labels[..., None])[..., 0].double() - lse
    adv = st["advantages"].double()
    adv = adv if adv.dim() == 2 else adv[:, None]
    ratio = (logp - st["old_logp"].double()).exp() if st["old_logp"] is not None else torch.ones_like(logp)
    bounded = ratio.clamp(1 - c["low"], 1 + c["high"])
    free = ratio * adv <= bounded * adv
    term = -torch.where(free, ratio, bounded) * adv
    slope = torch.where(free, -ratio * adv, 0.0)
    clipped = (~free).double()
    kl = torch.zeros_like(logp)
    log_ratio = ref_lse = None
    if c["kl"] == "full":
        y = st["ref_logits"]
        _, _, ref_lse = _softmax_parts(y)
        # log p - log q over the vocabulary; its mean is small against its terms and summed in 64 bits
        log_ratio = x.float() - y.float()
        kl = (e * log_ratio).sum(-1, dtype=torch.float64) / total[..., 0] - (lse - ref_lse)
    elif st["ref_logits"] is not None or st["ref_logp"] is not None:
        ref = _token_logp(st["ref_logits"], labels) if st["ref_logits"] is not None else st["ref_logp"].double()
        d = logp - ref
        if c["kl"] == "kl":
            kl, more = d, torch.ones_like(d)
        elif c["kl"] == "abs":
            kl, more = d.abs(), d.sign()
        elif c["kl"] == "mse":
            kl, more = 0.5 * d * d, d
        else:
            kl, more = torch.expm1(-d) + d, -torch.expm1(-d)
        slope = slope + c["kl_beta"] * more
    if c["reduce"] == "token":
        weight = mask / mask.sum()
    else:
        length = mask.sum(-1, keepdim=True)
        weight = mask / length.clamp(min=1.0) / (length > 0).sum()
    share = mask / mask.sum()
    got = {"loss": ((term + c["kl_beta"] * kl) * weight).sum().float(), "logp": (logp * (mask != 0)).float(),
           "kl": (kl * share).sum().float(), "clipped": (clipped * share).sum().float()}
    if c["train"]:
        scaled = weight * st["scale"].double()
        if log_ratio is None:
            got["grad"] = _logits_grad(e, total, labels, slope * scaled, x.dtype)
        else:
            pull = log_ratio.sub_((lse - ref_lse + kl).float()[..., None]).mul_((c["kl_beta"] * scaled).float()[..., None])
            pull.sub_((slope * scaled).float()[..., None]).mul_(e).mul_((1 / total).float())
            pull.scatter_add_(-1, labels[..., None], (slope * scaled).float()[..., None])
            got["grad"] = pull.to(x.dtype)
    return got


def _router_plain(st, c):
    x, k = st["logits"].detach(), c["k"]
    t, n_exp = x.shape
    # the largest logits are the largest probabilities; equal ones go to the lower index
    experts = x.sort(dim=-1, descending=True, stable=True).indices[:, :k].contiguous()
    e, total, lse = _softmax_parts(x)
    p = e / total.float()
    chosen = p.gather(-1, experts)
    mass = chosen.sum(-1, keepdim=True)
    weights = chosen / mass if k > 1 else chosen
    hits = (experts[..., None] == torch.arange(n_exp, device=x.device)).sum(1)
    counts = hits.sum(0)
    keep = torch.ones(t, 1, device=x.device, dtype=torch.bool) if st["mask"] is None else st["mask"][:, None]
    kept = keep.sum().double()
    load = (hits * keep).sum(0).double() / (kept * k)
    balance = n_exp * (load * ((p * keep).sum(0, dtype=torch.float64) / kept)).sum()
    z = (lse.square() * keep[:, 0]).sum() / kept
    got = {"weights": weights, "experts": experts, "counts": counts, "balance": balance.float(), "z": z.float()}
    if c["train"]:
        inner = (weights * st["dw"]).sum(-1, keepdim=True) if k > 1 else 0.0
        into = (st["dw"] - inner) / mass if k > 1 else st["dw"]
        dp = (st["dloss"].double() * n_exp / kept * load).float()[None] * keep
        dp = dp.scatter_add(-1, experts, into)
        grad = p * (dp - (dp * p).sum(-1, keepdim=True))
        grad = grad + p * ((2.0 * st["dz"].double() / kept) * lse[:, None]).float() * keep
        got["grad"] = grad.to(x.dtype)
    return got


# ---------------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    x = st["logits"].detach()
    if case["op"] == "router":
        return _router_exact(case, st, x.double())
    keep = st["mask"].nonzero(as_tuple=True)                                  # rows outside have neither value nor gradient
    rows = x[keep].double()
    norm = torch.logsumexp(rows, -1, keepdim=True)
    at = st["labels"][keep][:, None]
    logp = (rows.gather(1, at) - norm)[:, 0]
    ref_rows = ref = None
    if st["ref_logits"] is not None:
        ref_rows = st["ref_logits"][keep].double()
        ref_rows -= torch.logsumexp(ref_rows, -1, keepdim=True)
        ref = ref_rows.gather(1, at)[:, 0]
    elif st["ref_logp"] is not None:
        ref = st["ref_logp"][keep].double()
    rows -= norm                                                              # log-probabilities of all words
    seq, n, s = keep[0], case["n"], case["s"]
    scale = float(st["scale"])
    by_seq = lambda v: torch.zeros(n, dtype=torch.float64, device=v.device).index_add_(0, seq, v)  # noqa: E731
    extra = None
    if case["op"] == "preference":
        policy = by_seq(logp)
        base = by_seq(ref) if ref is not None else torch.zeros_like(policy)
        margin = policy - base
        h, eps = n // 2, case["smoothing"]
        z = case["beta"] * (margin[:h] - margin[h:])
        sure = torch.nn.functional.logsigmoid
        got = {"loss": -((1 - eps) * sure(z) + eps * sure(-z)).mean(), "logp": policy, "ref_logp": base}
        dz = -((1 - eps) * torch.sigmoid(-z) - eps * torch.sigmoid(z)) * case["beta"] / h
        slope = (torch.cat([dz, -dz]) * scale + st["dlogp"].double())[seq]
    else:
        adv = st["advantages"].double()
        adv = adv[keep] if adv.dim() == 2 else adv[seq]
        r = torch.exp(logp - st["old_logp"][keep].double()) if st["old_logp"] is not None else torch.ones_like(logp)
        cap = torch.clamp(r, 1 - case["low"], 1 + case["high"])
        term, outside = -torch.minimum(r * adv, cap * adv), r * adv > cap * adv
        slope = torch.where(outside, torch.zeros_like(r), -r * adv)
        d = torch.zeros_like(logp) if ref is None else logp - ref
        kl = torch.zeros_like(logp)
        if case["kl"] == "full":
            extra = rows - ref_rows
            kl = (rows.exp() * extra).sum(-1)
            extra -= kl[:, None]
        elif ref is not None:
            kl = {"kl": d, "abs": d.abs(), "mse": d ** 2 / 2, "k3": torch.exp(-d) - 1 + d}[case["kl"]]
            rise = {"kl": torch.ones_like(d), "abs": d.sign(), "mse": d, "k3": 1 - torch.exp(-d)}[case["kl"]]
            slope = slope + case["kl_beta"] * rise
        length = by_seq(torch.ones_like(logp))
        share = torch.full_like(logp, 1.0 / logp.numel())
        weight = share if case["reduce"] == "token" else 1.0 / (length[seq] * (length > 0).sum())
        whole = torch.zeros(n, s, dtype=torch.float64, device=x.device)
        whole[keep] = logp
        got = {"loss": ((term + case["kl_beta"] * kl) * weight).sum(), "logp": whole, "kl": (kl * share).sum(),
               "clipped": (outside.double() * share).sum()}
        slope = slope * weight * scale
        if extra is not None:
            extra *= (case["kl_beta"] * weight * scale)[:, None]
    if case["train"]:
        prob = rows.exp_()
        change = prob * (-slope[:, None] if extra is None else extra.sub_(slope[:, None]))
        change.scatter_add_(1, at, slope[:, None])
        grad = torch.zeros(n, s, x.shape[-1], dtype=torch.float64, device=x.device)
        grad[keep] = change
        got["grad"] = grad
    return got


def _router_exact(case, st, x):
    k, t = case["k"], x.shape[0]
    p = torch.softmax(x, -1)
    lse = torch.logsumexp(x, -1)
    order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :k]
    top = p.gather(1, order)
    w = top / top.sum(-1, keepdim=True) if k > 1 else top
    keep = torch.ones(t, dtype=torch.float64, device=x.device) if st["mask"] is None else st["mask"].double()
    n_kept = keep.sum()
    taken = torch.zeros_like(p).scatter_(1, order, 1.0)
    f = (taken * keep[:, None]).sum(0) / (n_kept * k)
    got = {"weights": w, "experts": None, "counts": None,
           "balance": x.shape[1] * (f * (p * keep[:, None]).sum(0) / n_kept).sum(), "z": (lse ** 2 * keep).sum() / n_kept}
    if case["train"]:
        dw = st["dw"].double()
        toward = (dw - (dw * w).sum(-1, keepdim=True)) / top.sum(-1, keepdim=True) if k > 1 else dw
        dp = torch.zeros_like(p).scatter_(1, order, toward)
        dp += float(st["dloss"]) * x.shape[1] * f[None] * keep[:, None] / n_kept
        got["grad"] = p * (dp - (dp * p).sum(-1, keepdim=True)) + p * (2 * float(st["dz"]) * lse * keep / n_kept)[:, None]
    return got


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = _DTYPES[case["dtype"]].itemsize
    if case["op"] == "router":
        cells, picks = case["tokens"] * case["experts"], case["tokens"] * case["k"]
        moved = cells * size + picks * 12 + case["experts"] * 8 + (case["tokens"] if case["padding"] else 0)
        if case["train"]:
            moved += cells * size + picks * 4
        return {"bytes": moved, "flops": cells * (5 + case["k"] + (6 if case["train"] else 0))}
    rows, v = _kept_rows(case), case["vocab"]
    streams = 2 if case["ref"] == "logits" else 1
    per_row = 12 + 4 * (case["ref"] == "logp") + (16 if case["op"] == "policy" else 0)
    moved = rows * (v * size * streams + per_row)
    cells = rows * v * 4 * streams
    if case["train"]:
        moved += case["n"] * case["s"] * v * size
        cells += rows * v * (7 if case.get("kl") == "full" else 4)
    return {"bytes": moved, "flops": cells}
