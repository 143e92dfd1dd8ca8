"""Distillation steps of a small model from a teacher's answers, end to end:

    python -m test1_amd.distillation_step [--steps N] [--words K] [--kind forward|reverse]

Two randomly initialised Llamas of a few layers are streamed through one GPU,
one after the other.  The teacher answers prompts (``SlideFSDP.sample_tokens``)
and leaves its largest log-probabilities of every token
(``SlideFSDP.top_logps``); the student takes steps on its divergence from them
(``SlideFSDP.forward(teacher=...)``).  One line for each step."""

from __future__ import annotations

import argparse

import torch

from . import SlideFSDP, SlideFSDPConfig


def make(layers: int, seed: int, device: str, lr: float):
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(seed)
    cfg = LlamaConfig(vocab_size=4096, hidden_size=512, intermediate_size=1024, num_hidden_layers=layers,
                      num_attention_heads=8, num_key_value_heads=4, max_position_embeddings=2048,
                      tie_word_embeddings=False)
    return SlideFSDP(LlamaForCausalLM(cfg), SlideFSDPConfig(device=device, lr=lr))


def main(argv=None) -> list:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--steps", type=int, default=4)
    p.add_argument("--rows", type=int, default=8)
    p.add_argument("--prompt", type=int, default=64)
    p.add_argument("--length", type=int, default=8, help="tokens that the teacher answers")
    p.add_argument("--words", type=int, default=32, help="words of the teacher for each token")
    p.add_argument("--kind", choices=("forward", "reverse"), default="forward")
    a = p.parse_args(argv)
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 4096, (a.rows, a.prompt), generator=g).to("cuda:0")
    teacher = make(6, 0, "cuda:0", 1e-4)
    for _ in range(a.length):
        token = teacher.sample_tokens(ids, torch.rand(a.rows, generator=g).to("cuda:0"), temperature=0.7, top_p=0.95)
        ids = torch.cat([ids, token.ids.unsqueeze(1)], dim=1)
    left = teacher.top_logps(ids, k=a.words)
    teacher.close()
    labels = ids.clone()
    labels[:, :a.prompt] = -100
    student = make(4, 1, "cuda:0", 1e-3)
    losses = []
    for i in range(a.steps):
        out = student(input_ids=ids, labels=labels, teacher=left, teacher_kind=a.kind)
        losses.append(float(out.loss.detach()))
        print(f"distillation step {i}: divergence {losses[-1]:.4f}", flush=True)
    student.close()
    return losses


if __name__ == "__main__":
    main()
