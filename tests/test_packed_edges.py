"""Packed-sequence operators at the edges of their range, against formulas in 64 bits."""

from __future__ import annotations

import pytest
import torch

from test_packed_ops import K, U, bf, norm_turned, rope_of, turned  # noqa: F401  (K is a fixture)

gpu = pytest.mark.gpu


# ---------------------------------------------------------------- gradients of the norms
def turned_size(x, rope):
    """The sum of the absolute values of the two terms of every rotated element, in 64 bits."""
    x = x.double()
    a, b = torch.zeros_like(x), torch.zeros_like(x)
    half = x.shape[-1] // 2
    first = torch.arange(x.shape[-1]) % 2 == 0 if rope is None or rope.interleaved else torch.arange(x.shape[-1]) < half
    a[..., first], b[..., ~first] = x[..., first], x[..., ~first]
    return turned(a, rope).abs() + turned(b, rope).abs()


def check_norm_gradients(K, q, k, qw, kw, rope, dq, dk, eps):
    grads = K.qk_norm_rope_bwd(q, k, qw, kw, rope, dq, dk, eps=eps)
    for x, w, dy, dx, dw in ((q, qw, dq, grads[0], grads[2]), (k, kw, dk, grads[1], grads[3])):
        xd, wd = x.double().requires_grad_(True), w.double().requires_grad_(True)
        want = torch.autograd.grad(norm_turned(xd, wd, rope, eps), (xd, wd), dy.double())
        xd = xd.detach()
        r = torch.rsqrt(xd.square().mean(-1, keepdim=True) + eps)
        n, g = xd * r, turned(dy, rope, -1.0)
        gw = g * w.double()
        # fp32: about ten roundings and one reciprocal root (two units) of terms of this size, then the type's own
        size = r * (gw.abs() + n.abs() * (gw * n).mean(-1, keepdim=True).abs()).amax(-1, keepdim=True)
        bound = 2.0 ** -19 * size + (U * want[0].abs() if x.dtype == torch.bfloat16 else 0.0) + 1e-37
        assert dx.dtype == x.dtype and ((dx.double() - want[0]).abs() <= bound).all()
        # fp32 sums over tokens and heads of terms (dy0 cos + dy1 sin) n: 2^-22 of the sum of absolute values covers a
        # tree of them
        assert dw.dtype == torch.float32
        assert ((dw.double() - want[1]).abs() <= 2.0 ** -18 * (turned_size(dy, rope) * n.abs()).sum((0, 1))).all()


def norm_inputs(tokens, heads, kv_heads, dim, dtype, size=1.0):
    return (bf(tokens, heads, dim, scale=size, dtype=dtype), bf(tokens, kv_heads, dim, scale=size, dtype=dtype),
            1 + 0.3 * bf(dim, dtype=torch.float32), bf(dim, dtype=torch.float32),
            bf(tokens, heads, dim, dtype=dtype), bf(tokens, kv_heads, dim, scale=3.0, dtype=dtype))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(19, 42, 42, 128), (300, 6, 1, 128), (5, 4, 4, 64),
                                                       (2500, 5, 3, 64), (1, 1, 0, 128)])
def test_norm_gradients_without_eps(K, tokens, heads, kv_heads, dim, dtype):  # noqa: F811
    """Head counts that leave a batch of loads part empty: the empty places have no norm at eps = 0."""
    torch.manual_seed(1)
    q, k, qw, kw, dq, dk = norm_inputs(tokens, heads, kv_heads, dim, dtype)
    check_norm_gradients(K, q, k, qw, kw, rope_of(tokens, dim, 3, True, "cuda"), dq, dk, 0.0)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size,eps", [(1e15, 1e-6), (1e17, 0.0), (1e-14, 1e-30), (1e-16, 0.0)])
def test_norm_gradients_of_large_and_small_rows(K, size, eps, dtype):  # noqa: F811
    """1 / rms and its square are fp32 numbers where its cube is not."""
    torch.manual_seed(2)
    q, k, qw, kw, dq, dk = norm_inputs(50, 4, 3, 128, dtype, size)
    check_norm_gradients(K, q, k, qw, kw, rope_of(50, 128, 3, False, "cuda"), dq, dk, eps)


@gpu
@pytest.mark.parametrize("eps", [1e-6, 1e-30])
def test_norm_gradients_of_zero_rows(K, eps):  # noqa: F811
    """A row of zeros has no direction: its gradient is w g / sqrt(eps), its part of the weights' is zero."""
    torch.manual_seed(3)
    q, k, qw, kw, dq, dk = norm_inputs(9, 3, 2, 64, torch.float32)
    q[4], k[:, 1] = 0.0, 0.0
    check_norm_gradients(K, q, k, qw, kw, None, dq, dk, eps)


# ---------------------------------------------------------------- layouts
def shifted(t, by=1):
    """The same values in contiguous memory that starts `by` elements past a 16-byte boundary."""
    flat = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
    return flat[by:].view(t.shape).copy_(t)


@gpu
@pytest.mark.parametrize("q_lens,heads,kv_heads", [([70, 33], 4, 2), ([1], 1, 1)])
def test_attention_of_contiguous_tensors_off_a_boundary(K, q_lens, heads, kv_heads):  # noqa: F811
    torch.manual_seed(4)
    plan = K.packed_plan(q_lens, heads=heads, kv_heads=kv_heads, head_dim=64, causal=True)
    n = plan.q_tokens
    q, k, v, do = bf(n, heads, 64), bf(n, kv_heads, 64), bf(n, kv_heads, 64), bf(n, heads, 64)
    o, lse = K.attention_packed_fwd(q, k, v, plan)
    want = (o, lse) + K.attention_packed_bwd(q, k, v, o, lse, do, plan)
    qs, ks, vs, os_, ds = (shifted(t) for t in (q, k, v, o, do))
    assert all(t.is_contiguous() and t.data_ptr() % 16 for t in (qs, ks, vs, os_, ds))
    got = K.attention_packed_fwd(qs, ks, vs, plan) + K.attention_packed_bwd(qs, ks, vs, os_, lse, ds, plan)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    K.check_status()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads", [(33, 3), (1, 1)])
def test_rotation_and_norms_of_contiguous_tensors_off_a_boundary(K, tokens, heads, dtype):  # noqa: F811
    torch.manual_seed(5)
    rope = rope_of(tokens, 64, 3, True, "cuda")
    q, k, qw, kw, dq, dk = norm_inputs(tokens, heads, heads, 64, dtype)
    qs, ks, dqs, dks = (shifted(t) for t in (q, k, dq, dk))
    want = K.rope_axes(q, k, rope) + K.qk_norm_rope(q, k, qw, kw, rope) + K.qk_norm_rope_bwd(q, k, qw, kw, rope, dq, dk)
    got = K.rope_axes(qs, ks, rope) + K.qk_norm_rope(qs, ks, qw, kw, rope) + \
        K.qk_norm_rope_bwd(qs, ks, qw, kw, rope, dqs, dks)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
