"""How training reaches the post-training losses and the router's losses, without a GPU: what a configuration's keys do or that they are
refused, and what online data has to bring."""
import pickle
import socket
import threading

import pytest
import torch

from common import make_args, run_distributed

MOE = {"moe_num_experts": 4, "moe_top_k": 2, "expert_interval": 1, "gpt_j_residual": False, "moe_loss_coeff": 0.1}


def _z_loss_step(rank, world, cfg, coeff, path):
    """``forward_step`` and its gradient: the loss, the gradient of the last layer's router weight, and what its router saw."""
    from gpt_neox_b200.initialize import initialize_megatron
    from gpt_neox_b200.models.moe import Router
    from gpt_neox_b200.training import forward_step, setup_model_and_optimizer
    from gpt_neox_b200.utils import Timers
    args = make_args(**{**cfg, "moe_z_loss_coeff": coeff, "global_num_gpus": world})
    args.configure_distributed_args()
    initialize_megatron(args)
    model, _, _, _ = setup_model_and_optimizer(args)
    routers = [m for m in model.module.modules() if isinstance(m, Router)]
    seen = []
    for r in routers:
        r.layer.register_forward_hook(lambda m, i, o: seen.append(i[0].detach().double()))
    text = torch.randint(1, 60, (2, args.seq_length + 1), generator=torch.Generator().manual_seed(1))
    loss, _ = forward_step(iter([{"text": text}]), model, args, Timers(), is_train=True)
    loss.backward()
    weight = routers[-1].layer.weight
    grad = weight.main_grad if getattr(weight, "main_grad", None) is not None and weight.grad is None else weight.grad
    torch.save({"loss": loss.detach().double(), "grad": grad.detach().double().clone(), "seen": seen,
                "weights": [r.layer.weight.detach().double() for r in routers]}, path)


@pytest.mark.parametrize("kind", ["megablocks", "deepspeed", "deepspeed dense"])
def test_z_loss_of_the_configuration_trains_the_router(kind, tmp_path):
    """The coefficient times the layers' mean of logsumexp^2 -- their mean or, for ``moe_type: deepspeed``, their sum, as the balance
    loss is taken -- enters the loss, and its gradient the router's weight."""
    cfg = {**MOE, "moe_type": kind.split()[0], "moe_use_residual": not kind.endswith("dense")}
    coeff, got = 0.05, []
    for i, c in enumerate((0.0, coeff)):
        run_distributed(_z_loss_step, 1, cfg, c, str(tmp_path / f"{i}.pt"))
        got.append(torch.load(tmp_path / f"{i}.pt"))
    off, on = got
    assert all(torch.equal(a, b) for a, b in zip(off["weights"], on["weights"]))
    z = torch.stack([(x.reshape(-1, w.shape[1]) @ w.t()).logsumexp(-1).square().mean() for x, w in zip(on["seen"], on["weights"])])
    share = z.sum() if kind.startswith("deepspeed") else z.mean()
    # losses of a few units and their differences in 32 bits: some roundings of 2^-24 each
    torch.testing.assert_close(on["loss"] - off["loss"], coeff * share, rtol=0, atol=2.0 ** -19)
    w = on["weights"][-1].requires_grad_()
    last = (on["seen"][-1].reshape(-1, w.shape[1]) @ w.t()).logsumexp(-1).square().mean() / (1 if kind.startswith("deepspeed") else len(z))
    want, = torch.autograd.grad(coeff * last, w)
    # a gradient in 32 bits is off by some hundred roundings of its largest terms, on either side of the difference
    torch.testing.assert_close(on["grad"] - off["grad"], want, rtol=0, atol=2.0 ** -15 * float(on["grad"].abs().max()))
    assert float(want.abs().max()) > 2.0 ** -12 * float(on["grad"].abs().max())


@pytest.mark.parametrize("change,words", [
    ({"train_impl": "dpo"}, "train_impl"), ({"train_impl": "reinforce"}, "train_impl"), ({"train_impl": "kto"}, "train_impl"),
    ({"train_impl": "rm"}, "train_impl"), ({"checkpoint_activations": True}, "checkpoint_activations"), ({"moe_loss_coeff": 0.0}, "moe_loss_coeff")])
def test_a_z_loss_that_would_not_train_is_refused(change, words):
    """Where a layer's auxiliary loss does not reach the router: objectives that leave it out, layers that run without a record first."""
    with pytest.raises(AssertionError, match=words):
        make_args(**{**MOE, "moe_z_loss_coeff": 0.01, **change})
    make_args(**{**MOE, **change})                                 # none asked for
    make_args(**{**MOE, "moe_z_loss_coeff": 0.01})


# ---------------------------------------------------------------------------------------------- online samples
BATCH = {"prefix": [5, 6], "completions": [[8, 9], [10, 11, 12]], "rewards": [1.0, 0.0], "logprobs": [[-0.5, -0.25], [-1.0, -2.0, -3.0]]}


def _online(*batches, **kw):
    """An ``OnlineDataset`` on a server that sends these batches."""
    from gpt_neox_b200.data.online_dataset import OnlineDataset
    srv = socket.socket()
    srv.bind(("127.0.0.1", 0))
    srv.listen(2)

    def serve():
        for batch in batches:
            conn, _ = srv.accept()
            conn.recv(64)
            conn.sendall(pickle.dumps(batch))
            conn.close()
    threading.Thread(target=serve, daemon=True).start()
    return OnlineDataset(num_samples=4, seq_length=6, leave_one_out=True, dataserver_ips="127.0.0.1", dataserver_ports=srv.getsockname()[1],
                         **kw)


@pytest.mark.parametrize("logprobs", [[[-0.5, -0.25]], [[-0.5, -0.25], [-1.0, -2.0, -3.0], [-1.0]]])
def test_online_log_probabilities_of_other_completions_are_refused(logprobs):
    """One list a completion: with fewer, samples whose rewards are in the baseline would be lost."""
    with pytest.raises(ValueError, match=f"log-probabilities of {len(logprobs)} completions"):
        _online({**BATCH, "logprobs": logprobs})[0]


def test_online_log_probabilities_may_come_as_arrays():
    import numpy as np
    ds = _online({**BATCH, "completions": [[8, 9], [10, 11]], "logprobs": np.array([[-0.5, -0.25], [-1.0, -2.0]])})
    assert ds[0]["old_logp"].tolist() == [0, 0, -0.5, -0.25, 0, 0, 0] and ds[1]["old_logp"].tolist() == [0, 0, -1, -2, 0, 0, 0]


def test_clipped_reinforce_names_what_its_samples_lack():
    """Samples without the sampler's log-probabilities: the error says which key asked for them, where the data comes in and where
    another loader's batch does."""
    from gpt_neox_b200.training import get_batch
    plain = {k: v for k, v in BATCH.items() if k != "logprobs"}
    with pytest.raises(ValueError, match="reinforce_clip.*logprobs"):
        _online(plain, needs_logprobs=True)[0]
    assert "old_logp" not in _online(plain)[0]
    assert "old_logp" in _online(BATCH, needs_logprobs=True)[0]
    args = make_args(train_impl="reinforce", reinforce_clip=0.2)
    text = torch.ones(2, 33, dtype=torch.long)
    whole = {"text": text, "label": text, "reward": torch.ones(2, 33), "raw_reward": torch.ones(2), "old_logp": torch.zeros(2, 33)}
    for key in ("label", "old_logp"):
        with pytest.raises(ValueError, match=f"reinforce_clip needs {key}"):
            get_batch(args, iter([{k: v for k, v in whole.items() if k != key}]))


@pytest.mark.parametrize("key,value", [("reinforce_clip_high", 0.3), ("reinforce_clip_high", 0.0), ("reinforce_sequence_mean", True)])
def test_options_of_the_clipped_objective_need_it(key, value):
    with pytest.raises(AssertionError, match=f"{key} needs reinforce_clip"):
        make_args(train_impl="reinforce", **{key: value})
    make_args(train_impl="reinforce", reinforce_clip=0.2, **{key: value})


def test_example_server_samples_from_the_policy_whose_log_probabilities_it_sends(monkeypatch):
    """With ``--logprobs`` the completions come from the whole distribution that the log-probabilities are of, not from its head."""
    import importlib.util
    import os
    from types import SimpleNamespace
    from common import ROOT
    spec = importlib.util.spec_from_file_location("server", os.path.join(ROOT, "post-training", "online_data_example_llama3.py"))
    server = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(server)
    own = torch.tensor
    monkeypatch.setattr(torch, "tensor", lambda *a, device=None, **kw: own(*a, **kw))
    seen = []
    sampler = server.Sampler.__new__(server.Sampler)
    sampler.tok = SimpleNamespace(eos_token_id=0)
    sampler.model = SimpleNamespace(generate=lambda ids, **kw: seen.append(kw) or torch.cat([ids, ids], 1))
    assert sampler.generate([3, 4], 1, 2) == [[3, 4]] and seen[0]["top_p"] == 0.95
    sampler.generate([3, 4], 1, 2, whole=True)
    assert seen[1]["top_p"] == 1.0 and seen[1]["top_k"] == 0 and seen[1]["temperature"] == 1.0 and seen[1]["do_sample"]


# ---------------------------------------------------------------------------------------------- arguments of the losses
def test_vocabularies_that_the_kernels_cannot_number_are_refused():
    from gpt_neox_b200.ops import policy_losses as PL
    many = torch.zeros(1, 1, 1).expand(2, 1, 2 ** 30)
    labels, mask = torch.zeros(2, 1, dtype=torch.long), torch.ones(2, 1)
    with pytest.raises(ValueError, match="words"):
        PL.preference_loss(many, labels, mask, 0.1)
    with pytest.raises(ValueError, match="words"):
        PL.policy_loss(many, labels, mask, mask)


def test_numbers_that_ask_for_a_gradient_are_refused():
    """The kernels take them as numbers: a gradient would be missing without a word."""
    from gpt_neox_b200.ops import policy_losses as PL
    x, labels, mask = torch.randn(2, 3, 5), torch.zeros(2, 3, dtype=torch.long), torch.ones(2, 3)
    learnt = torch.tensor(0.1, requires_grad=True)
    for call in (lambda t: PL.preference_loss(x, labels, mask, t), lambda t: PL.preference_loss(x, labels, mask, 0.1, label_smoothing=t),
                 lambda t: PL.policy_loss(x, labels, mask, mask, ref_logp=mask, kl_beta=t),
                 lambda t: PL.policy_loss(x, labels, mask, mask, clip_low=t), lambda t: PL.policy_loss(x, labels, mask, mask, clip_high=t)):
        with pytest.raises(ValueError, match="constant"):
            call(learnt)
        call(learnt.detach())
