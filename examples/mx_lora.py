"""Train LoRA adapters over a base frozen in 4 bits, then decode with them.

    python examples/mx_lora.py [--hidden 1024] [--ffn 2816] [--steps 30] [--fmt mxfp4]

A gated feed-forward block (the three projections of a decoder layer) is taken
from 16 bits to 4 with an adapter beside each projection; the adapters learn to
follow a slightly changed copy of the block while every linear keeps its input in 8 bits
for the backward pass; the trained block then runs one token at a time, as in
decoding.  Prints the losses, what the weights and the kept activations take, and
the time of a step and of a token.
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from probe_b200 import MXLoRALinear  # noqa: E402


class FeedForward(nn.Module):
    def __init__(self, hidden: int, ffn: int):
        super().__init__()
        kw = {"bias": False, "device": "cuda", "dtype": torch.bfloat16}
        self.gate, self.up, self.down = nn.Linear(hidden, ffn, **kw), nn.Linear(hidden, ffn, **kw), nn.Linear(ffn, hidden, **kw)

    def forward(self, x):
        return self.down(F.silu(self.gate(x)) * self.up(x))


def to_mx_lora(block: nn.Module, rank: int, scale: float, fmt: str) -> nn.Module:
    """Every ``nn.Linear`` child replaced by an ``MXLoRALinear``: A random, B zero, as LoRA starts."""
    for name, lin in list(block.named_children()):
        if isinstance(lin, nn.Linear):
            a = torch.randn(rank, lin.in_features) / math.sqrt(lin.in_features)
            setattr(block, name, MXLoRALinear(lin, a, torch.zeros(lin.out_features, rank), scale, fmt))
    return block


def timed(fn, n: int) -> float:
    """Milliseconds a call."""
    fn()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(n):
        fn()
    end.record()
    end.synchronize()
    return begin.elapsed_time(end) / n


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser()
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--ffn", type=int, default=2816)
    ap.add_argument("--rank", type=int, default=16)
    ap.add_argument("--tokens", type=int, default=2000)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--fmt", default="mxfp4", choices=("mxfp4", "nvfp4"))
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    teacher = FeedForward(args.hidden, args.ffn)
    student = FeedForward(args.hidden, args.ffn)
    student.load_state_dict(teacher.state_dict())
    with torch.no_grad():  # what the adapters have to learn: a change of low rank in each projection
        for lin in (teacher.gate, teacher.up, teacher.down):
            n, k = lin.weight.shape
            lin.weight += (torch.randn(n, 4, device="cuda") @ torch.randn(4, k, device="cuda")).mul_(0.5 / k).to(lin.weight)
    dense_bytes = sum(p.numel() * 2 for p in student.parameters())
    student = to_mx_lora(student, args.rank, 2.0, args.fmt)
    mx_bytes = sum(m.weight.nbytes for m in student.children())

    x = torch.randn(args.tokens, args.hidden, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        want = teacher(x).float()
    opt = torch.optim.Adam(student.parameters(), lr=1e-3)
    losses, kept = [], 0

    def pack(t):
        nonlocal kept
        kept += t.numel() * t.element_size() if t.dtype == torch.uint8 else 0
        return t

    def step():
        nonlocal kept
        opt.zero_grad(set_to_none=True)
        kept = 0
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            loss = (student(x).float() - want).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())

    for _ in range(args.steps):
        step()
    ms = timed(step, 5)
    token = x[:1]
    with torch.no_grad():
        us = 1e3 * timed(lambda: student(token), 50)
    first, last = float(losses[0]), float(losses[args.steps - 1])
    inputs = args.tokens * (2 * args.hidden + args.ffn) * 2
    print(f"loss {first:.5f} -> {last:.5f} in {args.steps} steps of {args.tokens} tokens, {ms:.2f} ms a step")
    print(f"weights {dense_bytes / 2**20:.1f} -> {mx_bytes / 2**20:.1f} MiB; inputs kept for the backward pass "
          f"{inputs / 2**20:.1f} -> {kept / 2**20:.1f} MiB; one token {us:.0f} us")
    return {"first": first, "last": last, "weight_bytes": mx_bytes, "dense_bytes": dense_bytes, "kept_bytes": kept,
            "input_bytes": inputs}


if __name__ == "__main__":
    main()
