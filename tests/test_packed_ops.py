"""Packed-sequence operators against formulas in 64 bits.

Rotation by positions on several axes, per-head norms of q and k with it, and
attention over packed sequences, forward and backward: the PyTorch kernel set
on the CPU (in float64, also against differences) and the native kernels on
the GPU.

Tolerances.  u = 2^-8 is the rounding error of bf16 (8 significand bits).
An output is rounded once; inside attention P and dS are rounded to bf16 once more, so an error is
bounded by u times the same sum over absolute values; delta is formed from the
rounded o.  Products of bf16 values accumulate in fp32, whose error is covered
by the 2^-11 added to u.
"""

from __future__ import annotations

import math

import pytest
import torch

from h3_a100.ops import AxisRope, TorchKernels

U = 2.0 ** -8 + 2.0 ** -11
R = TorchKernels()
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from h3_a100.ops.native import NativeKernels

    kernels = NativeKernels(torch.device("cuda", 0), wait_limit_s=2.0)
    yield kernels
    kernels.check_status()


# ---------------------------------------------------------------- formulas in 64 bits
def dense(q, k, v, plan, scale=None, do=None):
    """o, lse, gradients and the sums over absolute values that bound their errors."""
    scale = plan.head_dim ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    group = plan.heads // plan.kv_heads
    out = {n: torch.zeros_like(q) for n in ("o", "o_abs", "dq", "dq_abs")}
    out |= {n: torch.zeros_like(k) for n in ("dk", "dv", "dk_abs", "dv_abs")}
    out["lse"] = torch.full((plan.heads, q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    out["s_abs"] = torch.zeros_like(out["lse"])
    q0 = k0 = 0
    for nq, nk in zip(plan.q_lens, plan.k_lens):
        for h in range(plan.heads if nq and nk else 0):
            rq, rk, g = slice(q0, q0 + nq), slice(k0, k0 + nk), h // group
            qs, ks, vs = q[rq, h], k[rk, g], v[rk, g]
            s = scale * qs @ ks.T
            see = torch.ones_like(s, dtype=torch.bool)
            if plan.causal:
                see = torch.arange(nk, device=q.device) - nk <= torch.arange(nq, device=q.device)[:, None] - nq
            s = torch.where(see, s, -math.inf)
            lse = torch.logsumexp(s, -1)
            p = torch.where(see, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None]), 0.0)
            o = p @ vs
            out["o"][rq, h], out["lse"][h, rq] = o, lse
            out["o_abs"][rq, h] = p @ vs.abs() + o.abs()
            out["s_abs"][h, rq] = scale * (qs.abs() @ ks.abs().T).amax(-1)
            if do is None:
                continue
            d = do[rq, h].double()
            dp = d @ vs.T
            ds = scale * p * (dp - (o * d).sum(-1, keepdim=True))
            ds_err = U * ds.abs() + scale * p * (U * (out["o_abs"][rq, h] * d.abs()).sum(-1, keepdim=True))
            out["dq"][rq, h] = ds @ ks
            out["dk"][rk, g] += ds.T @ qs
            out["dv"][rk, g] += p.T @ d
            out["dq_abs"][rq, h] = ds_err @ ks.abs()
            out["dk_abs"][rk, g] += ds_err.T @ qs.abs()
            out["dv_abs"][rk, g] += U * (p.T @ d.abs())
        q0, k0 = q0 + nq, k0 + nk
    return out


def within(got, want, bound):
    err = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all()
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert worst <= 0.0, f"over the bound by {worst:.3g} (largest error {err.max().item():.3g})"
    # Roundings are as often up as down: in the 2-norm they stay near u itself.
    assert err.norm() <= 2 * U * want.norm() + 1e-9, f"norm of the error {(err.norm() / want.norm()).item():.3g}"


def rope_of(tokens, head_dim, axes, interleaved, device="cpu", pairs=None):
    """Axes of 31 x 24 x 42-like extents; fractional positions on the first one."""
    g = torch.Generator().manual_seed(tokens + head_dim)
    half = head_dim // 2
    if pairs is None:
        pairs = tuple(half // axes + (a < half % axes) for a in range(axes))
    pos = torch.rand(tokens, len(pairs), generator=g) * 42
    pos[:, 1:] = pos[:, 1:].floor()
    freqs = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in pairs]).float()
    return AxisRope(pos.to(device), freqs.to(device), pairs, interleaved)


def turned(x, rope, sign=1.0):
    """The rotation as complex products, in 64 bits."""
    x = x.double()
    half = x.shape[-1] // 2
    angle = torch.zeros(x.shape[0], half, dtype=torch.float64, device=x.device)
    if rope is not None:
        at = 0
        for a, n in enumerate(rope.pairs):
            angle[:, at:at + n] = rope.positions[:, a:a + 1].double() * rope.freqs[at:at + n].double()
            at += n
    turn = torch.polar(torch.ones_like(angle), sign * angle)[:, None]
    if rope is None or rope.interleaved:
        return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], half, 2)) * turn).reshape(x.shape)
    z = torch.complex(x[..., :half], x[..., half:]) * turn
    return torch.cat([z.real, z.imag], -1)


def norm_turned(x, w, rope, eps):
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    return turned(n * w, rope)


# ---------------------------------------------------------------- the PyTorch kernel set, CPU
LENGTHS = [([7], None, 4, 4, False), ([5, 0, 1, 12], None, 4, 2, True), ([1, 3], [9, 3], 6, 2, True),
           ([4, 2], [2, 0], 3, 1, True), ([6, 3], [5, 11], 2, 2, False)]


@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,causal", LENGTHS)
def test_torch_attention_is_the_formula(q_lens, k_lens, heads, kv_heads, causal):
    torch.manual_seed(1)
    plan = R.packed_plan(q_lens, k_lens, heads=heads, kv_heads=kv_heads, head_dim=8, causal=causal)
    q, do = (torch.randn(plan.q_tokens, heads, 8, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(plan.k_tokens, kv_heads, 8, dtype=torch.float64) for _ in range(2))
    o, lse = R.attention_packed_fwd(q, k, v, plan)
    grads = R.attention_packed_bwd(q, k, v, o, lse, do, plan)
    want = dense(q, k, v, plan, do=do)
    # 64-bit sums of fewer than 100 terms of size one
    for got, name in zip((o, lse) + grads, ("o", "lse", "dq", "dk", "dv")):
        torch.testing.assert_close(got, want[name], rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("causal", [False, True])
def test_attention_gradients_against_differences(causal):
    torch.manual_seed(2)
    plan = R.packed_plan([4, 1, 3], [4, 5, 2], heads=4, kv_heads=2, head_dim=6, causal=causal)
    q, do = (torch.randn(8, 4, 6, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(11, 2, 6, dtype=torch.float64) for _ in range(2))
    o, lse = R.attention_packed_fwd(q, k, v, plan)
    grads = R.attention_packed_bwd(q, k, v, o, lse, do, plan)
    step = 1e-5       # central differences: error step^2 ~ 1e-10 and 1e-16 / step ~ 1e-11
    for x, g in zip((q, k, v), grads):
        for i in torch.randperm(x.numel())[:40].tolist():
            flat = x.view(-1)
            old, values = flat[i].item(), []
            for s in (step, -step):
                flat[i] = old + s
                values.append((R.attention_packed_fwd(q, k, v, plan)[0] * do).sum().item())
            flat[i] = old
            assert abs((values[0] - values[1]) / (2 * step) - g.reshape(-1)[i].item()) < 1e-7


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("pairs", [(4,), (1, 2, 1), (0, 3), (1, 0, 1, 1)])
def test_torch_norm_rope_is_the_formula(pairs, interleaved):
    torch.manual_seed(3)
    rope = rope_of(9, 8, 0, interleaved, pairs=pairs)
    q, k = torch.randn(9, 3, 8, dtype=torch.float64), torch.randn(9, 2, 8, dtype=torch.float64)
    qw, kw = torch.randn(8, dtype=torch.float64), torch.randn(8, dtype=torch.float64)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    for got, x in zip(R.rope_axes(q, k, rope), (q, k)):
        torch.testing.assert_close(got, turned(x, rope), rtol=1e-12, atol=1e-12)
    for got, x in zip(R.rope_axes(*R.rope_axes(q, k, rope), rope, inverse=True), (q, k)):
        torch.testing.assert_close(got, x, rtol=1e-12, atol=1e-12)
    leaves = [t.clone().requires_grad_(True) for t in (q, qw, k, kw)]
    y = norm_turned(leaves[0], leaves[1], rope, 1e-6), norm_turned(leaves[2], leaves[3], rope, 1e-6)
    want = torch.autograd.grad(y, leaves, (dq, dk))
    out = R.qk_norm_rope(q, k, qw, kw, rope, eps=1e-6)
    grads = R.qk_norm_rope_bwd(q, k, qw, kw, rope, dq, dk, eps=1e-6)
    for got, ref in zip(out + grads, y + (want[0], want[2], want[1], want[3])):
        torch.testing.assert_close(got, ref.detach(), rtol=1e-10, atol=1e-10)


def test_descriptions_refuse():
    with pytest.raises(ValueError, match="positions must be"):
        AxisRope(torch.zeros(4, 2), torch.zeros(4), (4,))
    with pytest.raises(ValueError, match="freqs must hold"):
        AxisRope(torch.zeros(4, 1), torch.zeros(3), (4,))
    with pytest.raises(ValueError, match="1 to 4 axes"):
        AxisRope(torch.zeros(4, 5), torch.zeros(5), (1, 1, 1, 1, 1))
    with pytest.raises(ValueError, match="fp32"):
        AxisRope(torch.zeros(4, 1, dtype=torch.float64), torch.zeros(4), (4,))
    with pytest.raises(ValueError, match="key lengths"):
        R.packed_plan([1, 2], [1], heads=1, kv_heads=1, head_dim=64)
    with pytest.raises(ValueError, match="multiple"):
        R.packed_plan([1], heads=3, kv_heads=2, head_dim=64)
    with pytest.raises(ValueError, match="negative"):
        R.packed_plan([-1], heads=2, kv_heads=2, head_dim=64)
    plan = R.packed_plan([3], heads=2, kv_heads=2, head_dim=8)
    with pytest.raises(ValueError, match="as planned"):
        R.attention_packed_fwd(torch.zeros(4, 2, 8), torch.zeros(3, 2, 8), torch.zeros(3, 2, 8), plan)


# ---------------------------------------------------------------- rotation and norms, GPU
def bf(*shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device="cuda") * scale).to(dtype)


def tolerance(want, dtype):
    """One rounding of the result, and the fp32 arithmetic of a few operations on values of its row."""
    row = want.abs().amax(-1, keepdim=True)
    return (U if dtype == torch.bfloat16 else 0.0) * want.abs() + 2.0 ** -20 * row + 1e-30


ROPES = [(1, 4, 4, 128, 3, True), (77, 3, 1, 64, 1, False), (601, 6, 2, 128, 3, False), (2600, 5, 5, 64, 4, True),
         (2371, 14, 2, 128, 2, True)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,axes,interleaved", ROPES)
def test_rotation(K, tokens, heads, kv_heads, dim, axes, interleaved, dtype):
    torch.manual_seed(4)
    rope = rope_of(tokens, dim, axes, interleaved, "cuda")
    qkv = bf(tokens, (heads + 2 * kv_heads) * dim, dtype=dtype)
    q = qkv[:, :heads * dim].view(tokens, heads, dim)
    k = qkv[:, heads * dim:(heads + kv_heads) * dim].view(tokens, kv_heads, dim)
    before = qkv.clone()
    for got, x in zip(K.rope_axes(q, k, rope), (q, k)):
        want = turned(x, rope)
        assert got.dtype == dtype and ((got.double() - want).abs() <= tolerance(want, dtype)).all()
    back = K.rope_axes(q, None, rope, inverse=True)
    want = turned(q, rope, -1.0)
    assert back[1] is None and ((back[0].double() - want).abs() <= tolerance(want, dtype)).all()
    assert torch.equal(qkv, before)


@gpu
def test_rotation_of_far_positions(K):
    """At position 10^6 the fp32 product's rounding alone would be 0.06 of a turn's radian."""
    pos = torch.tensor([[1e6 + 0.25], [123456.5], [3e7], [0.0], [-5e5]], device="cuda")
    freqs = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    rope = AxisRope(pos, freqs, (64,))
    q = bf(5, 2, 128, dtype=torch.float32)
    want = turned(q, rope)
    assert ((K.rope_axes(q, q, rope)[1].double() - want).abs() <= tolerance(want, torch.float32)).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,axes,interleaved", ROPES)
def test_norm_rope_forward_and_gradients(K, tokens, heads, kv_heads, dim, axes, interleaved, dtype):
    torch.manual_seed(5)
    rope = rope_of(tokens, dim, axes, interleaved, "cuda") if axes != 2 else None
    q, k = bf(tokens, heads, dim, dtype=dtype), bf(tokens, kv_heads, dim, scale=0.2, dtype=dtype)
    qw, kw = 1 + 0.3 * bf(dim, dtype=torch.float32), bf(dim, dtype=torch.float32)
    dq, dk = bf(tokens, heads, dim, dtype=dtype), bf(tokens, kv_heads, dim, scale=3.0, dtype=dtype)
    out = K.qk_norm_rope(q, k, qw, kw, rope, eps=1e-5)
    grads = K.qk_norm_rope_bwd(q, k, qw, kw, rope, dq, dk, eps=1e-5)
    again = K.qk_norm_rope_bwd(q, k, qw, kw, rope, dq, dk, eps=1e-5)
    leaves = [t.double().requires_grad_(True) for t in (q, qw, k, kw)]
    y = norm_turned(leaves[0], leaves[1], rope, 1e-5), norm_turned(leaves[2], leaves[3], rope, 1e-5)
    want = torch.autograd.grad(y, leaves, (dq.double(), dk.double()))
    for got, ref in zip(out + grads[:2], (y[0].detach(), y[1].detach(), want[0], want[2])):
        assert got.dtype == dtype and ((got.double() - ref).abs() <= tolerance(ref, dtype)).all()
    for got, ref, x, dy, w in ((grads[2], want[1], q, dq, qw), (grads[3], want[3], k, dk, kw)):
        # fp32 sums over tokens and heads: 2^-22 of the sum of absolute values covers a tree of them
        n = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-5)
        size = (turned(dy, rope, -1.0) * n).abs().sum((0, 1))
        assert got.dtype == torch.float32 and ((got.double() - ref).abs() <= 2.0 ** -18 * size).all()
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@gpu
def test_norm_rope_layouts_and_empty_calls(K):
    torch.manual_seed(6)
    rope = rope_of(33, 128, 3, True, "cuda")
    q, k = bf(4, 33, 128).transpose(0, 1), bf(33, 2, 136)[..., 4:132]      # heads first; unaligned rows
    w = bf(128)
    got = K.qk_norm_rope(q, k, w, w, rope)
    want = K.qk_norm_rope(q.contiguous(), k.contiguous(), w, w, rope)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    grads = K.qk_norm_rope_bwd(q, k, w, w, rope, q[:1].expand(33, -1, -1), k, eps=1e-6)
    want = K.qk_norm_rope_bwd(q.contiguous(), k.contiguous(), w, w, rope, q[:1].repeat(33, 1, 1), k.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    zero = rope_of(0, 128, 3, True, "cuda")
    out = K.qk_norm_rope(bf(0, 4, 128), bf(0, 2, 128), w, w, zero)
    assert out[0].shape == (0, 4, 128) and out[1].shape == (0, 2, 128)
    grads = K.qk_norm_rope_bwd(bf(0, 4, 128), bf(0, 2, 128), w, w, zero, bf(0, 4, 128), bf(0, 2, 128))
    assert not grads[2].any() and not grads[3].any()
    # a row of zeros has no direction: the norm gives zeros, the gradient stays finite
    out = K.qk_norm_rope(torch.zeros_like(q), torch.zeros_like(k), w, w, rope)
    assert not out[0].any() and not out[1].any()


@gpu
def test_norm_rope_refusals(K):
    q, k, w = bf(4, 2, 128), bf(4, 2, 128), bf(128)
    rope = rope_of(4, 128, 3, True, "cuda")
    bad = [
        ((bf(4, 2, 96), bf(4, 2, 96), bf(96), bf(96), None), "head_dim"),
        ((q.half(), k.half(), w, w, rope), "bf16 or fp32"),
        ((q, k.float(), w, w, rope), "one type"),
        ((q, bf(5, 2, 128), w, w, rope), "tokens"),
        ((q, k, bf(64), w, rope), "q_weight"),
        ((q, k, w, w.float(), rope), "one type"),
        ((q, k, w, w, rope_of(5, 128, 3, True, "cuda")), "positions"),
        ((q, k, w, w, rope_of(4, 128, 3, True, "cpu")), "positions"),
        ((bf(4, 2, 64), bf(4, 2, 64), bf(64), bf(64), rope), "more rotation pairs"),
    ]
    for args, message in bad:
        with pytest.raises(RuntimeError, match=message):
            K.qk_norm_rope(*args)
    with pytest.raises(RuntimeError, match="heads of q and k"):
        K.qk_norm_rope_bwd(q, k, w, w, rope, bf(4, 3, 128), k)


# ---------------------------------------------------------------- attention, GPU
ATTENTION = [
    # lengths at, below and above a tile; one token; nothing
    ([128], None, 2, 2, False), ([1], None, 1, 1, True), ([129, 127, 1, 0, 256], None, 2, 2, True),
    ([300, 65], None, 3, 3, False), ([513, 40], None, 8, 2, True), ([1000, 7, 333], None, 4, 1, True),
    # groups that do not divide 128
    ([200, 100], None, 6, 2, True), ([150, 31], None, 7, 1, False), ([40], None, 65, 1, True),
    # other keys than queries: new tokens over older keys, cross attention, rows that see nothing, no keys
    ([1, 1, 5], [700, 1, 300], 8, 2, True), ([3, 130], [257, 511], 4, 4, False), ([300, 200], [100, 201], 4, 2, True),
    ([5, 140, 3], [0, 20, 0], 2, 1, True), ([0, 9], [200, 0], 2, 2, False),
    # key ranges that are split over blocks
    ([1, 2], [9000, 5000], 8, 2, True), ([400], [6000], 2, 2, False), ([2, 300], [7000, 4100], 7, 1, True),
    # few rows over many keys, some sequences without keys or queries
    ([1, 3, 0, 2], [9000, 0, 77, 6000], 8, 2, True), ([1, 1], [5000, 3001], 4, 4, False), ([9], [4000], 14, 2, True),
]


def make(plan, scale=1.0):
    qkv = bf(plan.q_tokens, (plan.heads + 2 * plan.kv_heads) * plan.head_dim, scale=scale)
    q = qkv[:, :plan.heads * plan.head_dim].view(plan.q_tokens, plan.heads, plan.head_dim)
    if plan.k_lens == plan.q_lens:
        k, v = qkv[:, plan.heads * plan.head_dim:].view(plan.q_tokens, 2, plan.kv_heads, plan.head_dim).unbind(1)
    else:
        k, v = (bf(plan.k_tokens, plan.kv_heads, plan.head_dim, scale=scale) for _ in range(2))
    return q, k, v


def check_forward(o, lse, want, dim):
    within(o, want["o"], U * want["o_abs"] + 1e-7)
    empty = want["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, empty) and not o.transpose(0, 1)[empty].any()
    # fp32 accumulation of dim products, exp2 and log2
    bound = 2.0 ** -24 * dim * want["s_abs"] + 2.0 ** -19
    assert ((lse.double() - want["lse"]).abs()[~empty] <= bound[~empty]).all()


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,causal", ATTENTION)
def test_attention(K, q_lens, k_lens, heads, kv_heads, causal, dim):
    torch.manual_seed(7)
    plan = K.packed_plan(q_lens, k_lens, heads=heads, kv_heads=kv_heads, head_dim=dim, causal=causal)
    q, k, v = make(plan)
    do = bf(plan.q_tokens, heads, dim)
    o, lse = K.attention_packed_fwd(q, k, v, plan)
    K.check_status()
    want = dense(q, k, v, plan, do=do)
    check_forward(o, lse, want, dim)
    grads = K.attention_packed_bwd(q, k, v, o, lse, do, plan)
    K.check_status()
    for got, name in zip(grads, ("dq", "dk", "dv")):
        within(got, want[name], want[name + "_abs"] + U * want[name].abs() + 1e-6)
    again = K.attention_packed_bwd(q, k, v, o, lse, do, plan)
    assert torch.equal(o, K.attention_packed_fwd(q, k, v, plan)[0])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    K.check_status()


@gpu
def test_attention_against_differences(K):
    """The gradient along a random direction against the change of the 64-bit forward."""
    torch.manual_seed(8)
    plan = K.packed_plan([70, 1, 200], [70, 30, 131], heads=4, kv_heads=2, head_dim=64, causal=True)
    q, k, v = make(plan)
    do = bf(plan.q_tokens, 4, 64)
    o, lse = K.attention_packed_fwd(q, k, v, plan)
    grads = K.attention_packed_bwd(q, k, v, o, lse, do, plan)
    for x, g, at in ((q, grads[0], 0), (k, grads[1], 1), (v, grads[2], 2)):
        way = torch.randn_like(x, dtype=torch.float64)
        values = []
        for step in (1e-4, -1e-4):
            moved = [t.double() for t in (q, k, v)]
            moved[at] = moved[at] + step * way
            values.append((dense(*moved, plan)["o"] * do.double()).sum())
        slope, ours = (values[0] - values[1]) / 2e-4, (g.double() * way).sum()
        # independent roundings of g: u |g| |way| in the 2-norm, three standard deviations and dS's, P's own
        assert abs(slope - ours) <= 6 * U * (g.double() * way).norm()


@gpu
@pytest.mark.parametrize("scale,size", [(0.05, 1.0), (1.0, 1.0), (1.0, 3.0), (0.088, 20.0)])
def test_attention_scales(K, scale, size):
    """Flat to one-hot rows: the running maximum jumps late and far."""
    torch.manual_seed(9)
    plan = K.packed_plan([260, 140], [700, 140], heads=4, kv_heads=2, head_dim=128, causal=True)
    q, k, v = make(plan, size)
    k[-1] *= 2.0
    o, lse = K.attention_packed_fwd(q, k, v, plan, scale=scale)
    want = dense(q, k, v, plan, scale)
    # scores of size s carry an fp32 error of 2^-24 dim s into the exponent, hence into every weight
    spread = 2.0 ** -24 * 128 * want["s_abs"].t()[..., None]
    assert ((o.double() - want["o"]).abs() <= (U + spread) * want["o_abs"] + 1e-6).all()
    assert ((lse.double() - want["lse"]).abs() <= 2.0 ** -24 * 128 * want["s_abs"] + 2.0 ** -19).all()
    K.check_status()


@gpu
def test_attention_keeps_sequences_apart(K):
    """NaN and infinities in the neighbours of a sequence, in the batch and past its end, do not reach it."""
    torch.manual_seed(10)
    lens = [70, 200, 1, 130]
    plan = K.packed_plan(lens, heads=6, kv_heads=2, head_dim=128, causal=False)
    q, k, v = (t.clone() for t in make(plan))
    do = bf(401, 6, 128)
    o, lse = K.attention_packed_fwd(q, k, v, plan)
    grads = K.attention_packed_bwd(q, k, v, o, lse, do, plan)
    for bad in (math.nan, math.inf):
        spoilt = [torch.full((n.shape[0] + 64, *n.shape[1:]), bad, dtype=n.dtype, device="cuda") for n in (q, k, v, do)]
        for s, n in zip(spoilt, (q, k, v, do)):
            s[:401] = n
            s[70:270] = bad
        views = [s[:401] for s in spoilt]
        o2, lse2 = K.attention_packed_fwd(*views[:3], plan)
        keep = torch.ones(401, dtype=torch.bool, device="cuda")
        keep[70:270] = False
        assert torch.equal(o2[keep], o[keep]) and torch.equal(lse2[:, keep], lse[:, keep])
        grads2 = K.attention_packed_bwd(*views[:3], o2, lse2, views[3], plan)
        for a, b in zip(grads2, grads):
            assert torch.equal(a[keep], b[keep])
    K.check_status()


@gpu
def test_attention_layouts(K):
    torch.manual_seed(11)
    plan = K.packed_plan([90, 45], heads=4, kv_heads=2, head_dim=64, causal=True)
    q, k, v = bf(4, 135, 64).transpose(0, 1), bf(135, 2, 72)[..., :64], bf(135, 2, 66)[..., 1:65]
    do = bf(1, 4, 64).expand(135, -1, -1)
    want_o, want_lse = K.attention_packed_fwd(q.contiguous(), k.contiguous(), v.contiguous(), plan)
    o, lse = K.attention_packed_fwd(q, k, v, plan)
    assert torch.equal(o, want_o) and torch.equal(lse, want_lse)
    want = K.attention_packed_bwd(q.contiguous(), k.contiguous(), v.contiguous(), o, lse, do.contiguous(), plan)
    fused = torch.full((135, 9 * 64), 7.0, dtype=torch.bfloat16, device="cuda")     # and a spare block of columns
    out = fused[:, :256].view(135, 4, 64), fused[:, 256:384].view(135, 2, 64), fused[:, 384:512].view(135, 2, 64)
    got = K.attention_packed_bwd(q, k, v, o, lse, do, plan, out=out)
    for a, b, c in zip(got, want, out):
        assert a.data_ptr() == c.data_ptr() and torch.equal(a, b)
    assert (fused[:, 512:] == 7.0).all()
    K.check_status()


@gpu
def test_attention_on_another_stream(K):
    torch.manual_seed(12)
    plan = K.packed_plan([1, 400], [5000, 400], heads=8, kv_heads=2, head_dim=128, causal=True)
    q, k, v = make(plan)
    do = bf(401, 8, 128)
    want = K.attention_packed_fwd(q, k, v, plan)
    want_grads = K.attention_packed_bwd(q, k, v, *want, do, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.attention_packed_fwd(q, k, v, plan)
        grads = K.attention_packed_bwd(q, k, v, *got, do, plan)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))


@gpu
def test_attention_in_a_graph(K):
    torch.manual_seed(13)
    plan = K.packed_plan([1] * 4, [3000, 9, 700, 6000], heads=8, kv_heads=2, head_dim=128, causal=True)
    q, k, v = make(plan)
    K.attention_packed_fwd(q, k, v, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = K.attention_packed_fwd(q, k, v, plan)
    q.copy_(bf(*q.shape))
    graph.replay()
    want = K.attention_packed_fwd(q, k, v, plan)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


@gpu
def test_attention_refusals(K):
    plan = K.packed_plan([4, 3], heads=4, kv_heads=2, head_dim=64, causal=True)
    q, k, v = bf(7, 4, 64), bf(7, 2, 64), bf(7, 2, 64)
    o, lse = K.attention_packed_fwd(q, k, v, plan)
    bad = [((q[:6], k, v), "q must be"), ((q, k.float(), v), "bf16"), ((q, k, v[:, :1]), "v must be"),
           ((q, k.cpu(), v), "k must be"), ((bf(7, 4, 128), k, v), "q must be")]
    for args, message in bad:
        with pytest.raises(RuntimeError, match=message):
            K.attention_packed_fwd(*args, plan)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="scale"):
            K.attention_packed_fwd(q, k, v, plan, scale=scale)
    with pytest.raises(ValueError, match="packed_plan"):
        K.attention_packed_fwd(q, k, v, R.packed_plan([7], heads=4, kv_heads=2, head_dim=64))
    with pytest.raises(RuntimeError, match="head_dim"):
        K.packed_plan([4], heads=4, kv_heads=2, head_dim=80)
    for args, message in (((o[:6], lse, q), "o must be"), ((o, lse[:, :6], q), "lse"), ((o, lse, q.float()), "bf16")):
        with pytest.raises(RuntimeError, match=message):
            K.attention_packed_bwd(q, k, v, *args, plan)
    with pytest.raises(RuntimeError, match="dq, dk and dv"):
        K.attention_packed_bwd(q, k, v, o, lse, q, plan, out=(q,))


@gpu
def test_out_views_and_their_refusals(K):
    torch.manual_seed(14)
    rope = rope_of(50, 64, 3, True, "cuda")
    q, k, dq, dk, w = bf(50, 4, 64), bf(50, 2, 64), bf(50, 4, 64), bf(50, 2, 64), bf(64)
    want = K.qk_norm_rope_bwd(q, k, w, w, rope, dq, dk)
    fused = torch.full((50, 7 * 64), 7.0, dtype=torch.bfloat16, device="cuda")
    out = fused[:, :256].view(50, 4, 64), fused[:, 256:384].view(50, 2, 64)
    got = K.qk_norm_rope_bwd(q, k, w, w, rope, dq, dk, out=out)
    assert got[0].data_ptr() == out[0].data_ptr() and all(torch.equal(a, b) for a, b in zip(got, want))
    assert (fused[:, 384:] == 7.0).all()
    for bad, message in (((out[0],), "dq and dk"), ((out[0], out[0]), "heads of q and k"),
                         ((out[0].float(), out[1]), "type"),
                         ((fused[:, 1:257].view(50, 4, 64), out[1]), "16-byte")):
        with pytest.raises(RuntimeError, match=message):
            K.qk_norm_rope_bwd(q, k, w, w, rope, dq, dk, out=bad)


@gpu
def test_checked_build_agrees(K):
    """The bounds-checked build gives the same bits and reports nothing."""
    try:
        from h3_a100 import _C_checked
    except ImportError:
        pytest.skip("bounds-checked extension not built (H3_CHECKED_BUILD=1 python setup.py build_ext --inplace)")
    from h3_a100.ops.native import NativeKernels

    checked = NativeKernels(torch.device("cuda", 0), wait_limit_s=2.0, extension=_C_checked)
    torch.manual_seed(15)
    for q_lens, k_lens, heads, kv, dim, causal in (([77, 1, 300], None, 6, 2, 128, True),
                                                   ([1, 2], [9000, 400], 8, 2, 64, True)):
        plan = K.packed_plan(q_lens, k_lens, heads=heads, kv_heads=kv, head_dim=dim, causal=causal)
        q, k, v = make(plan)
        do = bf(plan.q_tokens, heads, dim)
        results = []
        for kernels in (K, checked):
            o, lse = kernels.attention_packed_fwd(q, k, v, plan)
            results.append((o, lse) + kernels.attention_packed_bwd(q, k, v, o, lse, do, plan))
            kernels.check_status()
        assert all(torch.equal(a, b) for a, b in zip(*results))
