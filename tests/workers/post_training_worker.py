"""Post-training steps on one GPU (launched by tests/test_policy_losses_gpu.py): ``dpo`` with a reference model, ``clipped``
REINFORCE, or ``moe`` with balance and z loss, in bf16.  The objective's loss and gradients agree with its plain statement on the same
model, and training steps run through the kernels.  Prints ``POST_TRAINING_OK``."""
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(os.path.dirname(HERE)))
sys.path.insert(0, os.path.dirname(HERE))


def main(kind):
    torch.cuda.set_device(0)
    from common import make_args
    from gpt_neox_b200.initialize import initialize_megatron
    from gpt_neox_b200.models import moe as M
    from gpt_neox_b200.ops import moe_ops as MO
    from gpt_neox_b200.ops import native
    from gpt_neox_b200.ops import policy_losses as PL
    from gpt_neox_b200.training import forward_step, setup_model_and_optimizer, train_step
    from gpt_neox_b200.utils import Timers
    more = {"dpo": {"train_impl": "dpo", "dpo_beta": 0.1},
            "clipped": {"train_impl": "reinforce", "reinforce_clip": 0.2, "reinforce_clip_high": 0.3, "kl_impl": "full"},
            "moe": {"moe_num_experts": 8, "moe_top_k": 2, "moe_z_loss_coeff": 0.01, "expert_interval": 1, "moe_glu": False}}[kind]
    args = make_args(hidden_size=256, num_attention_heads=4, num_layers=2, seq_length=128, max_position_embeddings=128,
                     precision="bfloat16", global_num_gpus=1, distributed_backend="nccl", zero_optimization={"stage": 1},
                     train_micro_batch_size_per_gpu=2, attention_config=[[["flash"], "all"]], train_iters=100, lr_decay_iters=100,
                     **more)
    args.configure_distributed_args()
    initialize_megatron(args)
    model, opt, sched, ref = setup_model_and_optimizer(args)
    g = torch.Generator().manual_seed(3)
    v = args.padded_vocab_size
    tok = lambda: torch.randint(1, v, (2, 129), generator=g)                      # noqa: E731
    if kind == "dpo":
        batch = {"pos": tok(), "neg": tok()}
        with torch.no_grad():                                                       # a policy that has moved from its reference
            for p in model.module.parameters():
                p.add_(torch.randn_like(p) * 0.002)
    elif kind == "clipped":
        text = tok()
        label = text.clone()
        label[:, :40] = -100
        batch = {"text": text, "label": label, "reward": torch.randn(2, 129, generator=g), "raw_reward": torch.rand(2, generator=g),
                 "old_logp": torch.full((2, 129), -5.5)}
        ref = None                                                                  # no reference: the clip alone
    else:
        batch = {"text": tok()}

    def it():
        while True:
            yield batch
    data = it()

    def loss_and_grads():
        for p in model.module.parameters():
            p.grad = None
            if getattr(p, "main_grad", None) is not None:
                p.main_grad.zero_()
        before = native.launch_count
        loss, _ = forward_step(data, model, args, Timers(), is_train=True, reference_model=ref)
        loss.backward()
        grads = [(p.main_grad if getattr(p, "main_grad", None) is not None and getattr(p, "grad_in_main", False) else p.grad)
                 for p in model.module.parameters()]
        return float(loss), torch.cat([x.float().reshape(-1) for x in grads if x is not None]), native.launch_count - before

    loss, grads, launches = loss_and_grads()
    own = PL._k, MO.router_kernel_ok
    PL._k = lambda *a: False
    import gpt_neox_b200.objectives as O
    O._k, kept = (lambda *a: False), O._k
    M.MO.router_kernel_ok = lambda *a: False
    plain, plain_grads, _ = loss_and_grads()
    PL._k, M.MO.router_kernel_ok = own
    O._k = kept
    # dpo: sums of at most 512 log-probabilities, each off by 2^-18 on either side, times beta.  The others are means of numbers of a
    # few units, with one rounding to bf16 (2^-8 of them) where the router hands its loss on
    bound = 4 * 512 * 2.0 ** -18 * (0.1 if kind == "dpo" else 1.0) if kind == "dpo" else 2.0 ** -7
    assert abs(loss - plain) <= bound, (loss, plain)
    # both backward passes start from logit gradients rounded to bf16 (2^-9 on average) and share every later kernel
    off = float((grads - plain_grads).norm() / plain_grads.norm())
    assert off <= 2.0 ** -6, off
    losses = []
    for _ in range(4):
        d, _ = train_step(args, Timers(), data, model, opt, sched, reference_model=ref)
        losses.append(float(d["lm_loss"]))
    assert all(l == l for l in losses) and launches > 0 and native.read_status() == 0, losses
    print("POST_TRAINING_OK", kind, loss, plain, off, losses)


if __name__ == "__main__":
    main(sys.argv[1])
