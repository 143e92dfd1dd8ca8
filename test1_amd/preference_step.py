"""Preference and policy fine-tuning steps of a small model, end to end:

    python -m test1_amd.preference_step [--steps N] [--checkpoint-format int8|fp8|none]

A randomly initialised Llama of a few layers is streamed through one GPU.  Its
log-probabilities before the first step are the reference policy's
(``SlideFSDP.token_logps``); then steps on ``preference_loss`` over pairs of
random answers, and steps on ``policy_loss`` with random advantages, run with
the decoders' checkpoints in 8 bits.  One line for each step."""

from __future__ import annotations

import argparse

import torch

from . import SlideFSDP, SlideFSDPConfig
from .alignment import policy_loss, preference_loss


def answers(pairs: int, prompt: int, length: int, vocab: int, device) -> tuple:
    """(ids, labels) of 2 ``pairs`` sequences: each pair shares a prompt, whose
    labels are ignored."""
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, vocab, (2 * pairs, prompt + length), generator=g)
    ids[pairs:, :prompt] = ids[:pairs, :prompt]
    labels = ids.clone()
    labels[:, :prompt] = -100
    return ids.to(device), labels.to(device)


def main(argv=None) -> list:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--steps", type=int, default=4, help="steps of each objective")
    p.add_argument("--pairs", type=int, default=4)
    p.add_argument("--length", type=int, default=192, help="tokens of an answer, behind a prompt of 64")
    p.add_argument("--checkpoint-format", choices=("int8", "fp8", "none"), default="int8")
    a = p.parse_args(argv)
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=4096, hidden_size=512, intermediate_size=1024, num_hidden_layers=4,
                      num_attention_heads=8, num_key_value_heads=4, max_position_embeddings=2048,
                      tie_word_embeddings=False)
    cfg._attn_implementation = "sdpa"
    dev = torch.device("cuda", torch.cuda.current_device())
    model = SlideFSDP(LlamaForCausalLM(cfg), SlideFSDPConfig(device=dev, lr=1e-4), wait_timeout=120,
                      checkpoint_format=None if a.checkpoint_format == "none" else a.checkpoint_format)
    ids, labels = answers(a.pairs, 64, a.length, cfg.vocab_size, dev)
    losses = []
    try:
        ref = model.token_logps(ids, labels=labels)
        for step in range(a.steps):
            out = model(input_ids=ids, labels=labels, objective=lambda lp, mask: preference_loss(lp, ref, mask, beta=0.1))
            margin = (out.result.chosen_rewards - out.result.rejected_rewards).mean()
            losses.append(out.loss.item())
            print(f"preference step {step}: loss {losses[-1]:.4f}, reward margin {margin.item():+.4f}", flush=True)
        old = model.token_logps(ids, labels=labels)
        advantages = torch.cat([torch.ones(a.pairs, device=dev), -torch.ones(a.pairs, device=dev)])
        for step in range(a.steps):
            out = model(input_ids=ids, labels=labels, objective=lambda lp, mask: policy_loss(
                lp, old, advantages, mask, ref_logps=ref, kl_coef=0.04, reduction="sequence"))
            losses.append(out.loss.item())
            print(f"policy step {step}: loss {losses[-1]:+.4f}, KL {out.result.kl.item():.5f}, "
                  f"clipped {out.result.clip_fraction.item():.3f}", flush=True)
        model.wait_for_updates()
    finally:
        model.close()
    return losses


if __name__ == "__main__":
    main()
