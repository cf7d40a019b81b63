"""A DoRA fine-tuning step on native operators from the norms to the optimizer.

Around the adapted projections (``layer.DoraLinear``) a training step needs the
normalisation in front of them, the loss behind the output projection and the
optimizer over the adapters; this module puts the native ones together on the
Llama-style decoder of ``model``:

  use_native_norms   swaps the model's RMS norms and layer norms for ``norms``
  causal_lm_loss     next-token loss from ``logprobs.token_logprobs``
  train_step         forward, backward and one ``optim.AdamW`` step

    python -m dorafactors_b200.finetune --layers 2 --steps 10 --state-bits 8

trains adapters on a repeated synthetic batch and prints each step's loss, the share of
its tokens that the model ranks first, and its time.
"""

from __future__ import annotations

import argparse

import torch
from torch import nn

from .logprobs import TokenLogprobs, token_logprobs
from .norms import LayerNorm, RMSNorm
from .optim import AdamW


def use_native_norms(model: nn.Module) -> int:
    """Swap every layer norm and RMS norm over the last dimension for the native module,
    which takes over the parameters themselves.  Returns how many were swapped."""
    swapped = 0
    for module in list(model.modules()):
        for name, child in list(module.named_children()):
            weight = getattr(child, "weight", None)
            if type(child) is nn.LayerNorm and len(child.normalized_shape) == 1:
                new = LayerNorm(child.normalized_shape[0], child.eps, elementwise_affine=False)
                new.weight, new.bias = child.weight, child.bias
            elif type(child).__name__.endswith("RMSNorm") and not isinstance(child, RMSNorm) and weight is not None:
                eps = getattr(child, "variance_epsilon", getattr(child, "eps", None))
                if eps is None or weight.ndim != 1:
                    continue
                new = RMSNorm(weight.shape[0], eps, elementwise_affine=False)
                new.weight = weight
            else:
                continue
            new.train(child.training)
            setattr(module, name, new)
            swapped += 1
    return swapped


def next_token_targets(labels: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """Each position's next label; the last one of a sequence is ignored.  The logits then need
    no slice, which would be a copy of them."""
    return torch.cat((labels[..., 1:], labels.new_full((*labels.shape[:-1], 1), ignore_index)), -1)


def causal_lm_loss(logits: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100, entropy_weight: float = 0.0,
                   top_k: int = 0) -> tuple[torch.Tensor, TokenLogprobs]:
    """Mean negative log probability of the next labels (less ``entropy_weight`` times the mean
    entropy), and the token log probabilities it comes from."""
    targets = next_token_targets(labels, ignore_index)
    out = token_logprobs(logits, targets, entropy=entropy_weight != 0.0, top_k=top_k, ignore_index=ignore_index)
    count = (targets != ignore_index).sum().clamp_min(1)
    total = out.logprobs.sum()
    if entropy_weight:
        total = total + entropy_weight * out.entropy.sum()
    return -total / count, out


def train_step(model: nn.Module, ids: torch.Tensor, optimizer: AdamW, labels: torch.Tensor | None = None,
               **loss_args) -> tuple[torch.Tensor, TokenLogprobs]:
    """One step on token ids [batch, length]; the labels are the ids unless given (-100: ignored)."""
    loss, out = causal_lm_loss(model(input_ids=ids).logits, ids if labels is None else labels, **loss_args)
    loss.backward()
    optimizer.step()
    optimizer.zero_grad(set_to_none=True)
    return loss.detach(), out


def main(argv=None) -> None:
    from . import _native
    from .model import add_dora, build_llama, llama_config

    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--ffn", type=int, default=3584)
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--rank", type=int, default=16)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--seq", type=int, default=512)
    ap.add_argument("--steps", type=int, default=10)
    ap.add_argument("--lr", type=float, default=1e-3)
    ap.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    ap.add_argument("--no-master", action="store_true", help="step on the bf16 adapters themselves")
    a = ap.parse_args(argv)
    config = llama_config(layers=a.layers, hidden=a.hidden, ffn=a.ffn, heads=a.hidden // 128, kv_heads=max(1, a.hidden // 512),
                          vocab=a.vocab, max_pos=a.seq)
    model = build_llama(config, "cuda")
    params = add_dora(model, r=a.rank, scaling=2.0)
    use_native_norms(model)
    opt = AdamW(params, lr=a.lr, state_bits=a.state_bits, master_weights=not a.no_master)
    gen = torch.Generator("cuda").manual_seed(0)
    ids = torch.randint(0, a.vocab, (a.batch, a.seq), device="cuda", generator=gen)
    targets = next_token_targets(ids)
    for step in range(a.steps):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        loss, out = train_step(model, ids, opt, top_k=1)
        end.record()
        first = (out.top_indices[..., 0] == targets)[targets != -100].float().mean()
        print(f"step {step}: loss {float(loss):.4f}, ranked first {float(first):.3f}, {begin.elapsed_time(end):.1f} ms")
    if _native.device_error(reset=True) != 0:
        raise SystemExit("device error word set")


if __name__ == "__main__":
    main()
