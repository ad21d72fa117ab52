"""Preference loss, clipped policy loss and the router with its losses without a GPU: their plain statements against formulas and
differences, what the entry points refuse, tensor parallelism on gloo ranks, and the training paths that call them."""
import pickle
import socket
import threading

import numpy as np
import pytest
import torch

from common import make_args, run_distributed, run_distributed_many

from gpt_neox_b200.ops import moe_ops as MO
from gpt_neox_b200.ops import policy_losses as PL


def _batch(n=4, s=6, v=23, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, s, v, dtype=dtype, generator=g)
    ref = x + 0.3 * torch.randn(n, s, v, dtype=dtype, generator=g)
    labels = torch.randint(0, v, (n, s), generator=g)
    mask = (torch.rand(n, s, generator=g) > 0.4).to(dtype)
    mask[0, 0] = 1
    return x.requires_grad_(), ref, labels, mask


def _logp(x, labels):
    return x.log_softmax(-1).gather(-1, labels[..., None])[..., 0]


@pytest.mark.parametrize("ref", ["none", "logp", "logits"])
@pytest.mark.parametrize("eps", [0.0, 0.2])
def test_preference_loss_formula_and_differences(ref, eps):
    x, y, labels, mask = _batch()
    kw = {"none": {}, "logp": {"ref_logp": _logp(y, labels)}, "logits": {"ref_logits": y}}[ref]
    out = PL.preference_loss(x, labels, mask, 0.3, label_smoothing=eps, **kw)
    p = (_logp(x, labels) * mask).sum(1)
    r = torch.zeros_like(p) if ref == "none" else (_logp(y, labels) * mask).sum(1)
    z = 0.3 * ((p[:2] - p[2:]) - (r[:2] - r[2:]))
    want = (-(1 - eps) * torch.log(torch.sigmoid(z)) - eps * torch.log(torch.sigmoid(-z))).mean()
    torch.testing.assert_close(out.loss, want, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(out.logp, p, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(out.ref_logp, r.detach(), rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda t: PL.preference_loss(t, labels, mask, 0.3, label_smoothing=eps, **kw)[:2], (x,))


@pytest.mark.parametrize("kl", ["none", "kl", "abs", "mse", "k3", "full"])
@pytest.mark.parametrize("reduce", ["token", "sequence"])
def test_policy_loss_formula_and_differences(kl, reduce):
    x, y, labels, mask = _batch(3, 5, 17, seed=1)
    mask[1] = 0                                                    # a sequence that keeps nothing
    g = torch.Generator().manual_seed(2)
    adv = torch.randn(3, 5, dtype=torch.float64, generator=g)
    logp = _logp(x, labels).detach()
    # away from the clip's bounds, so that differences see one branch
    old = logp - torch.tensor([-0.6, -0.1, 0.1, 0.6, 0.05], dtype=torch.float64)
    kw = dict(old_logp=old, clip_low=0.2, clip_high=0.4, kl="k3" if kl == "none" else kl, kl_beta=0.3, reduce=reduce)
    if kl != "none":
        kw["ref_logits"] = y
    out = PL.policy_loss(x, labels, mask, adv, **kw)
    r = (_logp(x, labels) - old).exp()
    term = -torch.minimum(r * adv, r.clamp(0.8, 1.4) * adv)
    d = _logp(x, labels) - _logp(y, labels)
    est = {"none": 0 * d, "kl": d, "abs": d.abs(), "mse": d * d / 2, "k3": torch.exp(-d) - 1 + d,
           "full": (x.softmax(-1) * (x.log_softmax(-1) - y.log_softmax(-1))).sum(-1)}[kl]
    rows = (term + 0.3 * est) * mask
    if reduce == "token":
        want = rows.sum() / mask.sum()
    else:
        want = (rows[[0, 2]].sum(1) / mask[[0, 2]].sum(1)).mean()
    torch.testing.assert_close(out.loss, want, rtol=1e-11, atol=1e-11)
    torch.testing.assert_close(out.kl, ((est * mask).sum() / mask.sum()).detach(), rtol=1e-11, atol=1e-11)
    torch.testing.assert_close(out.clipped, ((r * adv > r.clamp(0.8, 1.4) * adv) * mask).sum() / mask.sum())
    torch.testing.assert_close(out.logp, logp * (mask != 0), rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda t: PL.policy_loss(t, labels, mask, adv, **kw).loss, (x,))


def test_masked_positions_do_not_matter():
    x, y, labels, mask = _batch(dtype=torch.float32)
    for kw in ({"ref_logits": y}, {"ref_logits": y, "kl": "full", "kl_beta": 0.1}):
        f = PL.policy_loss if "kl" in kw else PL.preference_loss
        args = (mask,) if "kl" in kw else (0.2,)
        clean = f(x, labels, mask, *args, **kw)
        want, = torch.autograd.grad(clean.loss, x)
        bad = x.detach().clone()
        bad[mask == 0] = float("nan")
        noise = y.clone()
        noise[mask == 0] = float("inf")
        other = torch.where(mask == 0, torch.full_like(labels, -100), labels)
        bad.requires_grad_()
        got = f(bad, other, mask, *args, **{**kw, "ref_logits": noise})
        grad, = torch.autograd.grad(got.loss, bad)
        assert torch.equal(got.loss, clean.loss) and torch.equal(grad, want) and not grad[mask == 0].any()


def test_policy_loss_on_policy_and_nothing_kept():
    x, _, labels, mask = _batch(dtype=torch.float32)
    adv = torch.randn(4)
    out = PL.policy_loss(x, labels, mask, adv)                     # without old_logp: minus the mean advantage
    torch.testing.assert_close(out.loss.detach(), -(adv[:, None] * mask).sum() / mask.sum(), rtol=1e-6, atol=1e-6)
    grad, = torch.autograd.grad(out.loss, x)
    want, = torch.autograd.grad(-(adv[:, None] * mask * _logp(x, labels)).sum() / mask.sum(), x)
    torch.testing.assert_close(grad, want, rtol=1e-5, atol=1e-7)
    for reduce in ("token", "sequence"):
        out = PL.policy_loss(x, labels, 0 * mask, adv, reduce=reduce)
        assert float(out.loss.detach()) == 0 and not torch.autograd.grad(out.loss, x)[0].any()


def test_refusals():
    x, y, labels, mask = _batch(dtype=torch.float32)
    bad = [
        (dict(logits=x[0]), "sequences, tokens, vocabulary"), (dict(logits=x[:0], labels=labels[:0], loss_mask=mask[:0]), "at least one"),
        (dict(logits=x[:3], labels=labels[:3], loss_mask=mask[:3]), "even number"), (dict(labels=labels[:, :3]), "labels is"),
        (dict(labels=labels.float()), "integers"), (dict(loss_mask=mask[:2]), "loss_mask is"), (dict(ref_logits=y[:, :2]), "ref_logits are"),
        (dict(ref_logits=y.half()), "ref_logits are"), (dict(ref_logits=y, ref_logp=mask), "not both"), (dict(ref_logp=mask[0]), "ref_logp is"),
        (dict(label_smoothing=1.0), "label_smoothing"), (dict(label_smoothing=-0.1), "label_smoothing"),
        (dict(ref_logits=x.detach().clone().requires_grad_()), "constant"), (dict(loss_mask=mask.clone().requires_grad_()), "constant"),
        (dict(logits=labels[..., None].expand(4, 6, 3)), "floating-point"),
    ]
    for change, words in bad:
        kw = dict(logits=x, labels=labels, loss_mask=mask, beta=0.1)
        kw.update(change)
        with pytest.raises(ValueError, match=words):
            PL.preference_loss(**kw)
    bad = [
        (dict(advantages=mask[:3]), "advantages are"), (dict(advantages=mask[..., None]), "advantages are"), (dict(old_logp=mask[:, :2]), "old_logp is"),
        (dict(kl="k2"), "kl is one of"), (dict(kl="full"), "needs ref_logits"), (dict(kl="full", ref_logp=mask), "needs ref_logits"),
        (dict(reduce="batch"), "reduce is"), (dict(clip_low=1.5), "clipped to"), (dict(clip_high=-0.1), "clipped to"),
        (dict(old_logp=mask.clone().requires_grad_()), "constant"), (dict(advantages=mask.clone().requires_grad_()), "constant"),
    ]
    for change, words in bad:
        kw = dict(logits=x, labels=labels, loss_mask=mask, advantages=mask)
        kw.update(change)
        with pytest.raises(ValueError, match=words):
            PL.policy_loss(**kw)
    z = torch.randn(5, 4)
    for args, words in (((z[0], 1), "tokens, experts"), ((z, 0), "top-k"), ((z, 5), "top-k"), ((z, 2, torch.ones(5)), "token_mask is bool"),
                        ((z, 2, torch.ones(4, dtype=torch.bool)), "token_mask is bool"), ((z.long(), 2), "floating-point")):
        with pytest.raises(ValueError, match=words):
            MO.balanced_router(*args)


@pytest.mark.parametrize("k", [1, 3])
def test_balanced_router_formula_and_differences(k):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 7, dtype=torch.float64, generator=g).requires_grad_()
    keep = torch.rand(40, generator=g) > 0.3
    out = MO.balanced_router(x, k, token_mask=keep)
    p, w, _, _ = MO.router_ref(x.detach(), k)
    torch.testing.assert_close(out.weights.detach().float(), w)
    hits = torch.zeros(40, 7, dtype=torch.float64).scatter_(1, out.experts, 1.0)
    assert torch.equal(out.counts, hits.sum(0).long())
    pk, hk = x.detach().softmax(-1)[keep], hits[keep]
    want = 7 * (hk.sum(0) / hk.sum() * pk.mean(0)).sum()
    torch.testing.assert_close(out.balance.detach(), want)
    torch.testing.assert_close(out.z.detach(), x.detach().logsumexp(-1)[keep].square().mean())
    assert torch.autograd.gradcheck(lambda t: [MO.balanced_router(t, k, token_mask=keep)[i] for i in (0, 3, 4)], (x,))
    even = torch.zeros(3, 4)
    assert MO.balanced_router(even, 2).experts.tolist() == [[0, 1]] * 3
    none = MO.balanced_router(x, k, token_mask=torch.zeros(40, dtype=torch.bool))
    assert float(none.balance.detach()) == 0 and float(none.z.detach()) == 0 and torch.equal(none.counts, out.counts)
    empty = MO.balanced_router(x[:0], k)
    assert float(empty.balance.detach()) == 0 and empty.counts.tolist() == [0] * 7


def _split_vocabulary(rank, world):
    from gpt_neox_b200.initialize import initialize_megatron
    args = make_args(global_num_gpus=world, model_parallel_size=world)
    args.configure_distributed_args()
    initialize_megatron(args)
    n, s, v = 4, 5, 16
    x, y, labels, mask = _batch(n, s, v * world, dtype=torch.float32, seed=4)
    labels[0, 0], labels[1, 1] = 0, v * world - 1
    mask[0, 1], labels[0, 1] = 0, -100
    share = lambda t: t.detach()[..., rank * v:(rank + 1) * v].clone()          # noqa: E731
    adv = torch.randn(n, generator=torch.Generator().manual_seed(1))
    wide = torch.where(labels < 0, 0, labels)
    for kl in ("k3", "full"):
        part = share(x).requires_grad_()
        out = PL.policy_loss(part, labels, mask, adv, old_logp=_logp(y, wide).detach(), ref_logits=share(y), kl=kl, kl_beta=0.2)
        grad, = torch.autograd.grad(out.loss, part)
        from unittest import mock
        with mock.patch.object(PL, "_tensor_parallel", lambda: (1, 0, None)):
            want = PL.policy_loss(x, labels, mask, adv, old_logp=_logp(y, wide).detach(), ref_logits=y, kl=kl, kl_beta=0.2)
        whole, = torch.autograd.grad(want.loss, x)
        torch.testing.assert_close(out.loss, want.loss, rtol=1e-5, atol=1e-6)
        torch.testing.assert_close(grad, share(whole), rtol=1e-4, atol=1e-6)
        part = share(x).requires_grad_()
        out = PL.preference_loss(part, labels, mask, 0.3, ref_logits=share(y))
        grad, = torch.autograd.grad(out.loss, part)
        with mock.patch.object(PL, "_tensor_parallel", lambda: (1, 0, None)):
            want = PL.preference_loss(x, labels, mask, 0.3, ref_logits=y)
        whole, = torch.autograd.grad(want.loss, x)
        torch.testing.assert_close(out.loss, want.loss, rtol=1e-5, atol=1e-6)
        torch.testing.assert_close(grad, share(whole), rtol=1e-4, atol=1e-6)


def test_losses_over_a_vocabulary_split_on_two_ranks():
    run_distributed(_split_vocabulary, 2)


# ---------------------------------------------------------------------------------------------- the paths that call them
def test_clipped_reinforce_objective():
    from gpt_neox_b200 import objectives as O
    x, y, labels, mask = _batch(dtype=torch.float32)
    rewards = torch.randn(4, 1).expand(4, 6)
    old = _logp(x, labels).detach() - 0.05
    loss, m = O.clipped_reinforce_loss(x, labels, mask, rewards, rewards[:, 0], old, 0.2, 0.3, kl_impl="k3", kl_beta=0.1, ref_logits=y,
                                       sequence_mean=True)
    want = PL.policy_loss(x, labels, mask, rewards, old_logp=old, ref_logits=y, clip_low=0.2, clip_high=0.3, kl="k3", kl_beta=0.1,
                          reduce="sequence")
    assert torch.equal(loss, want.loss) and torch.equal(m["kl"], want.kl) and set(m) == {"logp", "reward", "reward_std", "clipped", "kl"}
    torch.testing.assert_close(m["logp"], (_logp(x, labels).detach() * mask).sum() / mask.sum(), rtol=1e-5, atol=1e-6)
    loss, m = O.clipped_reinforce_loss(x, labels, mask, rewards, rewards[:, 0], old, 0.2)
    assert "kl" not in m and torch.isfinite(loss)
    # the plain objective knows the same estimate
    d = _logp(x, labels) - _logp(y, labels)
    loss, _ = O.reinforce_loss(x, labels, mask, rewards, rewards[:, 0], kl_impl="k3", kl_beta=0.1, ref_logits=y)
    want = ((-_logp(x, labels) * rewards + 0.1 * (torch.exp(-d) - 1 + d)) * mask).sum(-1).div(mask.sum()).mean()
    torch.testing.assert_close(loss, want, rtol=1e-5, atol=1e-6)


def test_online_samples_carry_the_samplers_log_probabilities():
    from gpt_neox_b200.data.online_dataset import OnlineDataset
    first = {"prefix": [5, 6], "completions": [[8, 9], [10, 11, 12, 13, 14, 15]], "rewards": [1.0, 0.0],
             "logprobs": [[-0.5, -0.25], [-1.0, -2.0, -3.0, -4.0, -5.0, -6.0]]}
    second = {**first, "logprobs": [[-0.5], [-1.0]]}
    srv = socket.socket()
    srv.bind(("127.0.0.1", 0))
    srv.listen(2)

    def serve():
        for batch in (first, second):
            conn, _ = srv.accept()
            conn.recv(64)
            conn.sendall(pickle.dumps(batch))
            conn.close()
    threading.Thread(target=serve, daemon=True).start()
    ds = OnlineDataset(num_samples=4, seq_length=6, leave_one_out=True, dataserver_ips="127.0.0.1", dataserver_ports=srv.getsockname()[1])
    a, b = ds[0], ds[1]
    assert a["old_logp"].tolist() == [0, 0, -0.5, -0.25, 0, 0, 0] and a["label"].tolist()[:4] == [-100, -100, 8, 9]
    assert np.array_equal(b["old_logp"], [0, 0, -1, -2, -3, -4, -5]) and b["old_logp"].dtype == np.float32
    with pytest.raises(ValueError, match="log-probabilities for"):
        ds[2]


def _clipped_training(rank, world, cfg):
    """``train_step`` with the clipped objective on batches of the online data's shape: finite metrics, and the gradient reaches
    the parameters."""
    from gpt_neox_b200.initialize import initialize_megatron
    from gpt_neox_b200.training import setup_model_and_optimizer, train_step
    from gpt_neox_b200.utils import Timers
    args = make_args(**{**cfg, "global_num_gpus": world})
    args.configure_distributed_args()
    initialize_megatron(args)
    model, opt, sched, ref = setup_model_and_optimizer(args)
    g = torch.Generator().manual_seed(7)
    mb, length, v = args.train_micro_batch_size_per_gpu, args.seq_length + 1, args.padded_vocab_size
    text = torch.randint(1, v, (mb, length), generator=g)
    label = text.clone()
    label[:, :9] = -100
    batch = {"text": text, "label": label, "reward": torch.randn(mb, length, generator=g), "raw_reward": torch.rand(mb, generator=g),
             "old_logp": torch.full((mb, length), -4.0)}

    def it():
        while True:
            yield batch
    source, before = it(), [p.detach().clone() for p in model.parameters()]
    for _ in range(3):
        d, _ = train_step(args, Timers(), source, model, opt, sched, reference_model=ref)
        assert all(float(v) == float(v) for v in d.values()), d
        assert {"clipped", "logp"} <= set(d) or any("clipped" in k for k in d), d
    assert any(not torch.equal(a, b) for a, b in zip(before, model.parameters()))


def test_clipped_reinforce_trains_end_to_end():
    base = {"train_impl": "reinforce", "reinforce_clip": 0.2, "train_micro_batch_size_per_gpu": 2}
    run_distributed_many((_clipped_training, 1, base),
                         (_clipped_training, 2, {**base, "model_parallel_size": 2, "reinforce_clip_high": 0.3, "reinforce_sequence_mean": True}))


def _router_z_loss(rank, world):
    from gpt_neox_b200.initialize import initialize_megatron
    from gpt_neox_b200.models.init_functions import get_init_methods
    from gpt_neox_b200.models.moe import ParallelMoE
    args = make_args(global_num_gpus=world, moe_num_experts=4, moe_top_k=2, moe_loss_coeff=0.1, moe_z_loss_coeff=0.02)
    args.configure_distributed_args()
    initialize_megatron(args)
    init, out_init = get_init_methods(args)
    moe = ParallelMoE(args, init, out_init, 4).float()
    x = torch.randn(10, 1, args.hidden_size)
    _, aux = moe(x)
    logits = moe.router.layer(x.reshape(10, -1))
    want = MO.balanced_router_ref(logits, 2)
    torch.testing.assert_close(0.1 * aux, 0.1 * want.balance + 0.02 * want.z, rtol=1e-5, atol=1e-6)
    args.moe_loss_coeff = 0.0
    with pytest.raises(ValueError, match="moe_loss_coeff"):
        ParallelMoE(args, init, out_init, 4)


def test_router_z_loss_joins_the_balance_loss():
    run_distributed(_router_z_loss, 1)


def test_more_tokens_than_the_kernels_number_are_refused():
    many = torch.zeros(1, 1, 1).expand(2 ** 15, 2 ** 15, 1)
    labels, mask = torch.zeros(1, 1, dtype=torch.long).expand(2 ** 15, 2 ** 15), many[..., 0]
    with pytest.raises(ValueError, match="fewer than"):
        PL.preference_loss(many, labels, mask, 0.1)
    with pytest.raises(ValueError, match="fewer than"):
        PL.policy_loss(many, labels, mask, mask)
    with pytest.raises(ValueError, match="fewer than"):
        MO.balanced_router(torch.zeros(1, 2).expand(2 ** 30, 2), 1)
