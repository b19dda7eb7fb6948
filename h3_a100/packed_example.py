"""Packed clips of different resolution through two attention layers, trained and served.

    python -m h3_a100.packed_example [--steps 20] [--device cuda|cpu] [--causal]

A batch of three clips (latent grids 8 x 12 x 20, 5 x 16 x 16 and 1 x 9 x 7, each
with its own text and audio tokens) is packed without padding.  A student whose
q/k norm weights are off is distilled into a teacher with the same frozen
projections: forward and backward of rotation, norms and attention every step.
Then, with a causal mask, new tokens are fed one at a time over the keys and
values of the tokens before them and compared with the whole prompt in one call.
"""

from __future__ import annotations

import argparse
import time

import torch

from .models.packed_attention import PackedSelfAttention
from .models.rope import axis_rope
from .ops import get_kernels

# (latent grid, text tokens, audio tokens)
CLIPS = (((8, 12, 20), 77, 120), ((5, 16, 16), 33, 80), ((1, 9, 7), 12, 0))


def tokens(clip) -> int:
    (f, h, w), text, audio = clip
    return f * h * w + text + audio


def build(kernels, device, *, hidden=512, heads=8, kv_heads=2, head_dim=64, layers=2, seed=0):
    torch.manual_seed(seed)
    dtype = torch.bfloat16 if device.type == "cuda" else torch.float32
    return torch.nn.ModuleList([PackedSelfAttention(hidden, heads, kv_heads, head_dim, kernels, dtype=dtype,
                                                    device=device) for _ in range(layers)])


def run(layers, x, plan, rope):
    for layer in layers:
        x = x + layer(x, plan, rope)
    return x


def train(kernels, device, *, steps: int, causal: bool, clips=CLIPS, hidden=512, lr=0.05, log=print) -> list[float]:
    teacher, student = (build(kernels, device, hidden=hidden) for _ in range(2))
    with torch.no_grad():
        for layer in teacher:
            layer.q_norm.mul_(1.5)
            layer.k_norm[::2] *= 0.5
    lens = [tokens(c) for c in clips]
    plan = student[0].plan(lens, causal=causal)
    rope = axis_rope(clips, student[0].head_dim, device=device)
    x = torch.randn(sum(lens), hidden, device=device).to(student[0].qkv_weight.dtype)
    with torch.no_grad():
        target = run(teacher, x, plan, rope).float()
    optim = torch.optim.Adam([p for p in student.parameters() if p.requires_grad], lr=lr)
    losses = []
    for step in range(steps):
        began = time.perf_counter()
        optim.zero_grad()
        loss = (run(student, x, plan, rope).float() - target).square().mean()
        loss.backward()
        optim.step()
        losses.append(loss.item())
        log(f"step {step}: loss {losses[-1]:.6f}  ({sum(lens)} tokens, {(time.perf_counter() - began) * 1e3:.1f} ms)")
    return losses


@torch.no_grad()
def serve(kernels, device, *, prompt=(40, 7, 129), new_tokens=4, hidden=512) -> float:
    """Largest difference between single new tokens over past keys and the whole prompt in one causal call."""
    layer = build(kernels, device, hidden=hidden, layers=1)[0]
    lens = [n + new_tokens for n in prompt]
    x = torch.randn(sum(lens), hidden, device=device).to(layer.qkv_weight.dtype)
    whole = layer(x, layer.plan(lens, causal=True))
    parts, wanted = x.split(lens), whole.split(lens)
    shape = (0, layer.kv_heads, layer.head_dim)
    past = tuple([torch.zeros(shape, dtype=x.dtype, device=device) for _ in lens] for _ in range(2))
    worst, done = 0.0, [0] * len(lens)
    for count in [list(prompt)] + [[1] * len(lens)] * new_tokens:
        seen = [a + b for a, b in zip(done, count)]
        y, past = layer(torch.cat([p[a:b] for p, a, b in zip(parts, done, seen)]),
                        layer.plan(count, seen, causal=True), past=past)
        for got, want, a, b in zip(y.split(count), wanted, done, seen):
            worst = max(worst, (got.float() - want[a:b].float()).abs().max().item())
        done = seen
    return worst


def main(argv=None) -> None:
    p = argparse.ArgumentParser()
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--causal", action="store_true")
    args = p.parse_args(argv)
    device = torch.device(args.device, 0) if args.device == "cuda" else torch.device(args.device)
    kernels = get_kernels("native", device)
    train(kernels, device, steps=args.steps, causal=args.causal)
    print(f"single tokens against the whole prompt: largest difference {serve(kernels, device):.2e}")
    if device.type == "cuda":
        kernels.check_status()


if __name__ == "__main__":
    main()
