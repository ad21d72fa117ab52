"""Which kernels a post-training step runs on one GPU (launched by tests/test_post_training_use_gpu.py): ``dpo`` with a reference model,
``clipped`` REINFORCE without one, ``reference``: clipped REINFORCE against a reference model, or ``moe`` with ``moe_type: deepspeed``
and a z loss, in bf16 over a vocabulary whose rows the clipped loss reads once.  The kernels run where they should and nowhere else,
and loss and gradients are those of the plain statements on the same model.  Prints ``KERNELS_OK``."""
import collections
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(os.path.dirname(HERE)))
sys.path.insert(0, os.path.dirname(HERE))

OWN = ("neox_loss_forward", "neox_policy_at_once", "neox_loss_backward", "neox_balanced_router", "neox_balanced_router_grad")


def main(kind):
    torch.cuda.set_device(0)
    from common import make_args
    import gpt_neox_b200.objectives as O
    from gpt_neox_b200.engine.engine import NeoXEngine
    from gpt_neox_b200.initialize import initialize_megatron
    from gpt_neox_b200.ops import moe_ops as MO
    from gpt_neox_b200.ops import native
    from gpt_neox_b200.ops import policy_losses as PL
    from gpt_neox_b200.training import forward_step, get_model, setup_model_and_optimizer, train_step
    from gpt_neox_b200.utils import Timers
    clipped = {"train_impl": "reinforce", "reinforce_clip": 0.2, "reinforce_clip_high": 0.3, "kl_impl": "k3"}
    more = {"dpo": {"train_impl": "dpo", "dpo_beta": 0.1}, "clipped": clipped, "reference": clipped,
            "moe": {"moe_num_experts": 8, "moe_top_k": 2, "moe_z_loss_coeff": 0.01, "expert_interval": 1, "moe_type": "deepspeed",
                    "moe_use_residual": False}}[kind]
    args = make_args(hidden_size=256, num_attention_heads=4, num_layers=2, seq_length=128, max_position_embeddings=128,
                     precision="bfloat16", global_num_gpus=1, distributed_backend="nccl", zero_optimization={"stage": 1},
                     train_micro_batch_size_per_gpu=2, attention_config=[[["flash"], "all"]], train_iters=100, lr_decay_iters=100,
                     make_vocab_size_divisible_by=8192, **more)
    args.configure_distributed_args()
    initialize_megatron(args)
    model, opt, sched, ref = setup_model_and_optimizer(args)
    g = torch.Generator().manual_seed(3)
    v = args.padded_vocab_size
    assert v == 8192
    tok = lambda: torch.randint(1, v, (2, 129), generator=g)                      # noqa: E731
    if kind in ("dpo", "reference"):
        with torch.no_grad():                                                       # a policy that has moved from its reference
            for p in model.module.parameters():
                p.add_(torch.randn_like(p) * 0.002)
    if kind == "dpo":
        batch = {"pos": tok(), "neg": tok()}
    elif kind == "moe":
        batch = {"text": tok()}
    else:
        text = tok()
        label = text.clone()
        label[:, :40] = -100
        batch = {"text": text, "label": label, "reward": torch.randn(2, 129, generator=g), "raw_reward": torch.rand(2, generator=g),
                 "old_logp": torch.full((2, 129), -9.0)}
        if kind == "reference":                                                     # which a caller hands to the step
            ref = NeoXEngine(get_model(neox_args=args), None, None, args)
        PL._REF_FIRST = 0                                                           # as a large batch has it
    calls, lib = collections.Counter(), native.lib()
    for name in OWN:
        def counted(*a, _name=name, _run=getattr(lib, name)):
            calls[_name] += 1
            return _run(*a)
        lib._cache[name] = counted

    def it():
        while True:
            yield batch
    data = it()

    def loss_and_grads():
        for p in model.module.parameters():
            p.grad = None
            if getattr(p, "main_grad", None) is not None:
                p.main_grad.zero_()
        calls.clear()
        loss, _ = forward_step(data, model, args, Timers(), is_train=True, reference_model=ref)
        loss.backward()
        grads = [(p.main_grad if getattr(p, "main_grad", None) is not None and getattr(p, "grad_in_main", False) else p.grad)
                 for p in model.module.parameters()]
        return float(loss.detach()), torch.cat([x.float().reshape(-1) for x in grads if x is not None]), dict(calls)

    loss, grads, ran = loss_and_grads()
    want = {"dpo": {"neox_loss_forward": 1, "neox_loss_backward": 1}, "clipped": {"neox_policy_at_once": 1, "neox_loss_backward": 1},
            "reference": {"neox_loss_forward": 1, "neox_policy_at_once": 1, "neox_loss_backward": 1},
            "moe": {"neox_balanced_router": 2, "neox_balanced_router_grad": 2}}[kind]
    assert ran == want, ran
    own = PL._k, O._k, MO.router_kernel_ok
    PL._k = O._k = MO.router_kernel_ok = lambda *a: False
    plain, plain_grads, ran = loss_and_grads()
    PL._k, O._k, MO.router_kernel_ok = own
    assert not ran, ran
    # dpo: sums of at most 512 log-probabilities, each off by 2^-18 on either side, times beta.  The others are means of numbers of a
    # few units, with one rounding to bf16 (2^-8 of them) where the router hands its loss on
    bound = 4 * 512 * 2.0 ** -18 * 0.1 if kind == "dpo" else 2.0 ** -7
    assert abs(loss - plain) <= bound, (loss, plain)
    # both backward passes start from logit gradients rounded to bf16 (2^-9 on average) and share every later kernel
    off = float((grads - plain_grads).norm() / plain_grads.norm())
    assert off <= 2.0 ** -6, off
    if kind == "moe":                                                               # and the z loss is part of them
        from gpt_neox_b200.models.moe import Router
        args.moe_z_loss_coeff = 0.0
        routers = [m for m in model.module.modules() if isinstance(m, Router)]
        for r in routers:
            r.z_share = 0.0
        _, without, ran = loss_and_grads()
        assert ran == {"neox_balanced_router": 2, "neox_balanced_router_grad": 2} and not torch.equal(grads, without), ran
    for _ in range(2):
        d, _ = train_step(args, Timers(), data, model, opt, sched, reference_model=ref)
        assert float(d["lm_loss"]) == float(d["lm_loss"])
    assert native.read_status() == 0
    print("KERNELS_OK", kind, loss, plain, off)


if __name__ == "__main__":
    main(sys.argv[1])
