"""The packed attention layer and its example: rotation helper, gradients, training, single tokens."""

from __future__ import annotations

import pytest
import torch

from h3_a100.models.packed_attention import PackedSelfAttention
from h3_a100.models.rope import axis_rope, rope_tables
from h3_a100.ops import TorchKernels, get_kernels
from h3_a100.ops.torch_kernels import Rope, rope_apply
from h3_a100.packed_example import serve, train

R = TorchKernels()
gpu = pytest.mark.gpu


def test_axis_rope_is_the_dit_rotation():
    """Each sample of a packed batch turns as the DiT's tables turn it alone."""
    torch.manual_seed(0)
    samples = [((3, 4, 5), 7, 11), ((1, 2, 2), 0, 0), ((2, 3, 3), 4, 6)]
    heads, dim = 2, 32
    lens = [f * h * w + t + a for (f, h, w), t, a in samples]
    q = torch.randn(sum(lens), heads, dim)
    got = R.rope_axes(q, None, axis_rope(samples, dim))[0]
    at = 0
    for (grid, text, audio), n in zip(samples, lens):
        cos, sin = rope_tables(grid, text, audio, dim)
        want = rope_apply(q[at:at + n].reshape(n, -1), Rope(cos, sin, dim, heads * dim, (0,)))
        # positions and frequencies are rounded to fp32 before their product: angles up to 5 rad differ by 1e-6
        torch.testing.assert_close(got[at:at + n].reshape(n, -1), want, rtol=0, atol=1e-5)
        at += n


@pytest.mark.parametrize("causal", [False, True])
def test_layer_gradients_against_autograd(causal):
    torch.manual_seed(1)
    hidden, heads, kv, dim, lens = 24, 4, 2, 8, [5, 9]
    layer = PackedSelfAttention(hidden, heads, kv, dim, R, dtype=torch.float64)
    layer.q_norm.data = torch.rand(dim, dtype=torch.float64) + 0.5
    layer.k_norm.data = torch.rand(dim, dtype=torch.float64) + 0.5
    samples = [((1, 1, 3), 2, 0), ((2, 2, 2), 1, 0)]
    rope = axis_rope(samples, dim)
    x = torch.randn(14, hidden, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(14, hidden, dtype=torch.float64)

    def plain(x, qw, kw):
        q, k, v = layer.split(x @ layer.qkv_weight.T + layer.qkv_bias)
        cos, sin = R._axis_tables(rope, dim, q)

        def normed(t, w):
            return R._turn(t * torch.rsqrt(t.square().mean(-1, keepdim=True) + layer.eps) * w, cos, sin, True)

        q, k = normed(q, qw), normed(k, kw)
        outs = []
        for a, b in ((0, 5), (5, 14)):
            qs = q[a:b].transpose(0, 1)
            ks, vs = (t[a:b].transpose(0, 1).repeat_interleave(heads // kv, 0) for t in (k, v))
            s = qs @ ks.transpose(1, 2) / dim ** 0.5
            if causal:
                s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool).triu(1), float("-inf"))
            outs.append((torch.softmax(s, -1) @ vs).transpose(0, 1))
        return torch.cat(outs).reshape(14, heads * dim) @ layer.out_weight.T + layer.out_bias

    plan = layer.plan(lens, causal=causal)
    y = layer(x, plan, rope)
    want = plain(x, layer.q_norm, layer.k_norm)
    inputs = (x, layer.q_norm, layer.k_norm)
    # The set's linear accumulates in fp32 after the product: 2^-24 of values of size one, summed over < 100 terms.
    torch.testing.assert_close(y, want, rtol=0, atol=2e-5)
    for got, ref in zip(torch.autograd.grad(y, inputs, dy), torch.autograd.grad(want, inputs, dy)):
        torch.testing.assert_close(got, ref, rtol=0, atol=2e-4)


@pytest.mark.parametrize("causal", [False, True])
def test_example_trains(causal):
    clips = (((2, 3, 4), 5, 3), ((1, 2, 2), 2, 0))
    losses = train(get_kernels("torch", torch.device("cpu")), torch.device("cpu"), steps=8, causal=causal, clips=clips,
                   hidden=64, log=lambda line: None)
    assert losses[-1] < 0.5 * losses[0]


def test_single_tokens_equal_the_whole_prompt():
    # the same fp32 sums over the same keys in another order
    assert serve(get_kernels("torch", torch.device("cpu")), torch.device("cpu"), prompt=(6, 1, 9), hidden=64) < 1e-5


@gpu
@pytest.mark.parametrize("causal", [False, True])
def test_example_trains_on_the_gpu(cuda, causal):
    kernels = get_kernels("native", cuda)
    before = kernels.launch_count()
    losses = train(kernels, cuda, steps=12, causal=causal, log=lambda line: None)
    assert losses[-1] < 0.5 * losses[0] and kernels.launch_count() > before
    # bf16 rounding of outputs of size one, after two roundings on the way
    assert serve(kernels, cuda) < 2.0 ** -5
    kernels.check_status()


@gpu
def test_layer_on_the_gpu_follows_the_plain_set(cuda):
    torch.manual_seed(3)
    kernels = get_kernels("native", cuda)
    layer = PackedSelfAttention(512, 8, 2, 64, kernels, device=cuda)
    samples = [((3, 5, 7), 20, 9), ((1, 1, 1), 0, 0), ((2, 9, 9), 3, 0)]
    lens = [f * h * w + t + a for (f, h, w), t, a in samples]
    rope = axis_rope(samples, 64, device=cuda)
    plan = layer.plan(lens, causal=True)
    x = torch.randn(sum(lens), 512, device=cuda).bfloat16().requires_grad_(True)
    dy = torch.randn(sum(lens), 512, device=cuda).bfloat16()
    y = layer(x, plan, rope)
    got = torch.autograd.grad(y, (x, layer.q_norm, layer.k_norm), dy)
    object.__setattr__(layer, "kernels", R)
    for name, t in list(layer.named_parameters()):
        t.data = t.data.float()
    xf = x.detach().float().requires_grad_(True)
    want_y = layer(xf, plan, rope)
    want = torch.autograd.grad(want_y, (xf, layer.q_norm, layer.k_norm), dy.float())
    # four roundings to bf16 (qkv, normed q/k, o, y) forward and as many again backward, 2^-8 each at most
    for a, b, roundings in ((y, want_y, 4), (got[0], want[0], 8), (got[1], want[1], 8), (got[2], want[2], 8)):
        a, b = a.detach().double(), b.detach().double()
        assert (a - b).norm() <= roundings * 2.0 ** -8 * b.norm()
    kernels.check_status()
