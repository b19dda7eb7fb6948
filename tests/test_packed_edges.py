"""Packed-sequence operators at the edges of their range, against formulas in 64 bits."""

from __future__ import annotations

import random

import pytest
import torch

from h3_a100.ops import AxisRope, PackedPlan, TorchKernels
from test_packed_ops import (K, U, bf, check_forward, dense, norm_turned, rope_of, turned,  # noqa: F401  (K: a fixture)
                             within)

_C = pytest.importorskip("h3_a100._C")
R = TorchKernels()
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


# ---------------------------------------------------------------- outputs in memory of the caller's
def _bytes(t):
    """Addresses of the elements of a view, one entry per place in its index space."""
    at = torch.tensor(t.storage_offset())
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return at.reshape(-1)


def _apart(out, ins=()):
    try:
        _C.check_apart(list(out), list(ins))
    except RuntimeError as e:
        assert "overlap" in str(e) or "over an input" in str(e)
        return False
    return True


def test_overlaps_are_what_sets_of_addresses_say():
    rng, flat, seen = random.Random(3), torch.zeros(4000), [0, 0, 0, 0]
    for _ in range(4000):
        views = []
        fused = rng.random() < 0.5
        row = rng.choice([16, 24, 40, 48])
        for _ in range(2):
            t, h, d = rng.randint(1, 6), rng.randint(1, 4), rng.choice([1, 2, 4, 8])
            strides = (row, rng.choice([d, 8, 12, 16])) if fused else (rng.randint(0, 40), rng.randint(0, 40))
            strides = strides if rng.random() < 0.7 else strides[::-1]
            views.append(flat.as_strided((t, h, d), (*strides, 1), rng.randint(0, 120)))
        a, b = (_bytes(v) for v in views)
        folded, shared = a.unique().numel() < a.numel(), bool(set(a.tolist()) & set(b.tolist()))
        assert _apart(views[:1]) == (not folded)
        if not folded:
            assert _apart(views[:1], views[1:]) == (not shared)
            seen[int(shared)] += 1
    assert min(seen[:2]) > 300


def test_layouts_of_models_are_apart():
    fused = torch.zeros(50, 8 * 64)
    q, k, v = fused[:, :256].view(50, 4, 64), fused[:, 256:384].view(50, 2, 64), fused[:, 384:].view(50, 2, 64)
    assert _apart([q, k, v]) and not _apart([q, k, k]) and not _apart([q, k], [fused])
    assert not _apart([fused[:, 32:288].view(50, 4, 64)], [q])
    turn = torch.zeros(50, 4, 3, 64)      # heads of q, k and v in turn
    assert _apart(turn.unbind(2)) and _apart([turn[:, :1, 0], turn[:, :, 1]], [turn[:, 2:3, 0]])
    first = torch.zeros(3, 4, 50, 64).transpose(1, 2)
    assert _apart(first.unbind(0)) and _apart([first[0, :, :2], first[0, :, 2:]])
    assert not _apart([first[0], first[0, 9:]])
    assert _apart([torch.zeros(0, 4, 64), torch.zeros(0, 4, 64)], [q])
    assert not _apart([torch.zeros(1, 4, 64).expand(50, -1, -1)])


def test_torch_gradients_into_inputs():
    """The PyTorch set writes after it has read."""
    torch.manual_seed(8)
    plan = R.packed_plan([5, 4], heads=2, kv_heads=2, head_dim=8, causal=True)
    q, k, v, do = (torch.randn(9, 2, 8, dtype=torch.float64) for _ in range(4))
    o, lse = R.attention_packed_fwd(q, k, v, plan)
    want = R.attention_packed_bwd(q, k, v, o, lse, do, plan)
    got = R.attention_packed_bwd(q, k, v, o, lse, do, plan, out=(q, k, v))
    assert all(a is b for a, b in zip(got, (q, k, v))) and all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="dq, dk and dv"):
        R.attention_packed_bwd(q, k, v, o, lse, do, plan, out=(q, k))


def test_torch_gradients_keep_the_type_of_out():
    torch.manual_seed(14)
    plan = R.packed_plan([6], heads=2, kv_heads=1, head_dim=8)
    q, k, v, do = (torch.randn(6, h, 8).bfloat16() for h in (2, 1, 1, 2))
    o, lse = R.attention_packed_fwd(q, k, v, plan)
    out = tuple(torch.empty(t.shape) for t in (q, k, v))
    R.attention_packed_bwd(q, k, v, o, lse, do, plan, out=out)
    short = R.attention_packed_bwd(q, k, v, o, lse, do, plan)
    assert all(torch.equal(a.bfloat16(), b) and not torch.equal(a, b.float()) for a, b in zip(out, short))


@gpu
def test_gradients_over_inputs_or_each_other_are_refused(K):  # noqa: F811
    plan = K.packed_plan([40, 9], heads=4, kv_heads=2, head_dim=64, causal=True)
    q, k, v, do = bf(49, 4, 64), bf(49, 2, 64), bf(49, 2, 64), bf(49, 4, 64)
    o, lse = K.attention_packed_fwd(q, k, v, plan)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    fused = bf(49, 8 * 64)
    for out, message in (((dq, dk, dk), "each other"), ((q, dk, dv), "over an input"), ((do, dk, dv), "over an input"),
                         ((o, dk, dv), "over an input"), ((dq, k, dv), "over an input"), ((dq, dk, v), "over an input"),
                         ((fused[:, :256].view(49, 4, 64), fused[:, 192:320].view(49, 2, 64), dv), "each other"),
                         ((dq, bf(50 * 64).as_strided((49, 2, 64), (64, 64, 1)), dv), "overlap itself")):
        with pytest.raises(RuntimeError, match=message):
            K.attention_packed_bwd(q, k, v, o, lse, do, plan, out=out)
    rope, w = rope_of(49, 64, 3, True, "cuda"), bf(64)
    dk_in = bf(49, 2, 64)
    for out, message in (((q, dk), "over an input"), ((dq, dk_in), "over an input"), ((do, dk), "over an input"),
                         ((fused[:, :256].view(49, 4, 64), fused[:, 192:320].view(49, 2, 64)), "each other"),
                         ((dq, bf(50 * 64).as_strided((49, 2, 64), (64, 64, 1))), "overlap itself")):
        with pytest.raises(RuntimeError, match=message):
            K.qk_norm_rope_bwd(q, k, w, w, rope, do, dk_in, out=out)


@gpu
def test_a_plan_dropped_while_another_stream_reads_it(K):  # noqa: F811
    """Its memory is not given to the next tensor of its own stream before the kernels are done."""
    torch.manual_seed(9)
    q_lens = [300, 41, 7]
    plan = K.packed_plan(q_lens, heads=4, kv_heads=2, head_dim=64, causal=True)
    q, k, v, do = bf(348, 4, 64), bf(348, 2, 64), bf(348, 2, 64), bf(348, 4, 64)
    want = K.attention_packed_fwd(q, k, v, plan)
    want += K.attention_packed_bwd(q, k, v, *want, do, plan)
    at, size = plan.blob.data_ptr(), plan.blob.numel()
    side, busy = torch.cuda.Stream(), torch.cuda.Event()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)      # about a tenth of a second
        got = K.attention_packed_fwd(q, k, v, plan)
        got += K.attention_packed_bwd(q, k, v, *got, do, plan)
        busy.record()
    del plan
    other = [torch.full((size,), -1, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert not busy.query(), "the side stream was not behind"
    assert all(t.data_ptr() != at for t in other)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    K.check_status()


# ---------------------------------------------------------------- scales
@gpu
def test_attention_scales_at_the_ends_of_fp32(K):  # noqa: F811
    """The kernels hold scale and scale * log2(e) in fp32: what is 0 or infinite there is refused."""
    torch.manual_seed(6)
    plan = K.packed_plan([40, 9], heads=2, kv_heads=1, head_dim=64, causal=True)
    q, k, v = bf(49, 2, 64), bf(49, 1, 64), bf(49, 1, 64)
    o, lse = K.attention_packed_fwd(q, k, v, plan, scale=1e-30)
    # scores of 1e-28: every visible key weighs the same
    seen = torch.cat([torch.arange(1, n + 1, device="cuda") for n in (40, 9)])
    assert ((lse.double() - seen.double().log()).abs() <= 2.0 ** -19).all()
    for scale in (1e-60, 1e39, 3e38):
        with pytest.raises(RuntimeError, match="scale"):
            K.attention_packed_fwd(q, k, v, plan, scale=scale)
        with pytest.raises(RuntimeError, match="scale"):
            K.attention_packed_bwd(q, k, v, o, lse, q, plan, scale=scale)


@gpu
def test_strided_positions_frequencies_and_weights(K):  # noqa: F811
    torch.manual_seed(7)
    rope = rope_of(21, 64, 3, True, "cuda")
    strided = AxisRope(rope.positions.t().contiguous().t(), rope.freqs.repeat_interleave(2)[::2], rope.pairs)
    assert strided.positions.stride() == (1, 21) and strided.freqs.stride() == (2,)
    q, k, qw, kw, dq, dk = norm_inputs(21, 3, 2, 64, torch.bfloat16)
    w2, w3 = torch.stack([qw, kw], 1).unbind(1)
    assert not w2.is_contiguous()
    want = K.rope_axes(q, k, rope) + K.qk_norm_rope(q, k, qw, kw, rope) + K.qk_norm_rope_bwd(q, k, qw, kw, rope, dq, dk)
    got = K.rope_axes(q, k, strided) + K.qk_norm_rope(q, k, w2, w3, strided) + \
        K.qk_norm_rope_bwd(q, k, w2, w3, strided, dq, dk)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rotation_is_a_copy():
    q, k = torch.randn(7, 3, 8).bfloat16(), torch.randn(7, 2, 8).bfloat16()
    for got, x in zip(R.rope_axes(q, k, None) + R.rope_axes(q, k, None, inverse=True), (q, k, q, k)):
        assert torch.equal(got, x) and got.data_ptr() != x.data_ptr()


@gpu
def test_no_rotation_is_a_copy_on_the_gpu(K):  # noqa: F811
    q, k = bf(7, 3, 64), bf(7, 2, 64)
    for got, x in zip(K.rope_axes(q, k, None) + K.rope_axes(q, k, None, inverse=True), (q, k, q, k)):
        assert torch.equal(got, x) and got.data_ptr() != x.data_ptr()


# ---------------------------------------------------------------- the bounds-checked build
@pytest.fixture(scope="module")
def checked():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    try:
        from h3_a100 import _C_checked
    except ImportError:
        pytest.skip("bounds-checked extension not built (H3_CHECKED_BUILD=1 python setup.py build_ext --inplace)")
    from h3_a100.ops.native import NativeKernels

    return NativeKernels(torch.device("cuda", 0), wait_limit_s=2.0, extension=_C_checked)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(1, 1, 1, 64), (77, 5, 3, 128), (2371, 14, 2, 64),
                                                       (9, 43, 42, 128)])
def test_checked_rotation_and_norms_agree(K, checked, tokens, heads, kv_heads, dim, dtype):  # noqa: F811
    torch.manual_seed(10)
    rope = rope_of(tokens, dim, 3, tokens % 2 == 0, "cuda")
    q, k, qw, kw, dq, dk = norm_inputs(tokens, heads, kv_heads, dim, dtype)
    results = []
    for kernels in (K, checked):
        fused = torch.zeros(tokens, (heads + kv_heads) * dim + 64, dtype=dtype, device="cuda")
        out = fused[:, 64:64 + heads * dim].view(q.shape), fused[:, 64 + heads * dim:].view(k.shape)
        results.append(kernels.rope_axes(q, k, rope) + kernels.qk_norm_rope(q, k, qw, kw, rope) +
                       kernels.qk_norm_rope_bwd(q, k, qw, kw, rope, dq, dk, out=out) + (fused,))
        kernels.check_status()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@gpu
def test_checked_build_reports_packed_operators(checked, monkeypatch):
    """With every allocation declared a head short, each kernel reports its last stores and skips them."""
    torch.manual_seed(11)
    dim = 128
    q, k, qw, kw, dq, dk = norm_inputs(33, 5, 3, dim, torch.bfloat16)
    plan = checked.packed_plan([33], heads=6, kv_heads=3, head_dim=dim, causal=True)
    split = checked.packed_plan([1], [9000], heads=6, kv_heads=3, head_dim=dim, causal=True)
    assert split.meta[9] > 0      # joins
    qa, do, ka, va = bf(33, 6, dim), bf(33, 6, dim), bf(33, 3, dim), bf(33, 3, dim)
    qs, ks, vs = bf(1, 6, dim), bf(9000, 3, dim), bf(9000, 3, dim)
    o, lse = checked.attention_packed_fwd(qa, ka, va, plan)
    grads = [torch.full_like(t, float("nan")) for t in (qa, ka, va)]
    norm_grads = [torch.full_like(t, float("nan")) for t in (q, k)]
    checked.check_status()

    def reported(call):
        monkeypatch.setenv("H3_BOUNDS_SHRINK", str(dim))
        call()
        torch.cuda.synchronize()
        monkeypatch.delenv("H3_BOUNDS_SHRINK")
        code = int(checked.status[0])
        checked.status.zero_()
        return code == 7

    assert reported(lambda: checked.rope_axes(q, None, None))
    assert reported(lambda: checked.qk_norm_rope(q, k, qw, kw))
    assert reported(lambda: checked.qk_norm_rope_bwd(q, k, qw, kw, None, dq, dk, out=norm_grads))
    assert reported(lambda: checked.attention_packed_fwd(qa, ka, va, plan))
    assert reported(lambda: checked.attention_packed_fwd(qs, ks, vs, split))
    assert reported(lambda: checked.attention_packed_bwd(qa, ka, va, o, lse, do, plan, out=grads))
    assert all(torch.isnan(t.view(-1, dim)[-1]).all() for t in grads + norm_grads)
    # (attention gradients of other rows may lack their delta and lse2, which were declared short too)
    assert all(not torch.isnan(t.view(-1, dim)[:-1]).any() for t in norm_grads)


# ---------------------------------------------------------------- every form of the attention kernels
JOINS, FEW, ITEMS, BEGIN, BLOCKS = 9, 19, 5, 6, 7      # places in a plan's meta


def forward_items(plan):
    ints, m = plan.blob.cpu(), plan.meta
    starts = ints[m[BEGIN]:m[BEGIN] + m[BLOCKS] + 1]
    return ints[m[ITEMS]:m[ITEMS] + 8 * int(starts[-1])].view(-1, 8).tolist()


def form_of(plan):
    two = any(item[1] > 128 // (plan.heads // plan.kv_heads) for item in forward_items(plan))
    return plan.meta[JOINS] > 0, bool(plan.meta[FEW]), two


# lengths, heads, key heads, and what they ask for: (split key ranges, few rows over many keys, two query tiles an item)
FORMS = [([70, 200, 1, 130], None, 6, 2, (False, False, False)),
         ([1031, 200, 777, 1299], None, 8, 8, (False, False, True)),
         ([130, 9, 300], [9001, 70, 4100], 4, 2, (True, False, False)),
         ([1290, 9, 300], [9001, 70, 4100], 13, 13, (True, False, True)),
         ([1, 3, 2], [9001, 257, 6001], 8, 2, (True, True, False))]


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,form", FORMS)
def test_every_form_keeps_sequences_apart(K, q_lens, k_lens, heads, kv_heads, form, causal, dim):  # noqa: F811
    """NaN or infinities in one sequence and past the end leave the others' bits alone."""
    torch.manual_seed(12)
    plan = K.packed_plan(q_lens, k_lens, heads=heads, kv_heads=kv_heads, head_dim=dim, causal=causal)
    assert form_of(plan) == form
    tensors = [bf(plan.q_tokens, heads, dim), bf(plan.k_tokens, kv_heads, dim), bf(plan.k_tokens, kv_heads, dim),
               bf(plan.q_tokens, heads, dim)]

    def run(q, k, v, do):
        o, lse = K.attention_packed_fwd(q, k, v, plan)
        grads = K.attention_packed_bwd(q, k, v, o, lse, do, plan)
        K.check_status()
        return (o, lse.t()) + grads

    want = run(*tensors)
    assert all(torch.isfinite(t).all() for t in want)
    spans = [slice(n[0], n[0] + n[1]) for n in (plan.q_lens, plan.k_lens)]
    for bad in (float("nan"), float("inf")):
        spoilt = []
        for t, at in zip(tensors, (0, 1, 1, 0)):
            room = torch.full((t.shape[0] + 300, *t.shape[1:]), bad, dtype=t.dtype, device="cuda")
            room[:t.shape[0]] = t
            room[spans[at]] = bad
            spoilt.append(room[:t.shape[0]])
        for got, ref, at in zip(run(*spoilt), want, (0, 0, 0, 1, 1)):
            keep = torch.ones(ref.shape[0], dtype=torch.bool, device="cuda")
            keep[spans[at]] = False
            assert torch.equal(got[keep], ref[keep])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,form", FORMS)
def test_second_query_tiles_see_no_fewer_key_tiles(q_lens, k_lens, heads, kv_heads, form, causal):
    """The loader fetches an item's keys for its second query tile; the first one's are among them."""
    lens = list(q_lens), list(q_lens if k_lens is None else k_lens)
    blob, meta = _C.packed_schedule(*lens, heads, kv_heads, 128, causal, 148)
    plan = PackedPlan(*lens, heads, kv_heads, 128, causal, blob, tuple(meta))
    assert form_of(plan) == form
    bt = 128 // (heads // kv_heads)
    for _, nq, _, nk, diag, _, _, _ in forward_items(plan):
        first, second = (-(-min(nk, max(0, n + diag)) // 128) for n in (min(bt, nq), nq))
        assert 0 < nq <= 2 * bt and first <= second


# ---------------------------------------------------------------- a long sequence
@gpu
@pytest.mark.parametrize("dim,causal", [(128, False), (128, True), (64, True)])
def test_attention_of_a_long_sequence(K, dim, causal):  # noqa: F811
    """The joint sequence of 37,730 tokens beside a short one, two heads on one, in blocks of queries."""
    torch.manual_seed(13)
    lens = [37730, 77]
    plan = K.packed_plan(lens, heads=2, kv_heads=1, head_dim=dim, causal=causal)
    q, k, v, do = bf(37807, 2, dim), bf(37807, 1, dim), bf(37807, 1, dim), bf(37807, 2, dim)
    o, lse = K.attention_packed_fwd(q, k, v, plan)
    grads = K.attention_packed_bwd(q, k, v, o, lse, do, plan)
    K.check_status()
    want = {}
    for at, n, step in ((0, 37730, 1290), (37730, 77, 77)):      # 37,730 is not a multiple of the step
        ks, vs = k[at:at + n], v[at:at + n]
        parts = []
        for i in range(0, n, step):
            rows = slice(at + i, at + min(i + step, n))
            part = PackedPlan((rows.stop - rows.start,), (n if not causal else rows.stop - at,), 2, 1, dim, causal)
            keys = part.k_lens[0]      # under a causal mask the last query of the block sees the last of these
            parts.append(dense(q[rows], ks[:keys], vs[:keys], part, do=do[rows]))
        for name in parts[0]:
            if name in ("dk", "dv", "dk_abs", "dv_abs"):
                total = torch.zeros(n, 1, dim, dtype=torch.float64, device="cuda")
                for p in parts:
                    total[:p[name].shape[0]] += p[name]
            else:
                total = torch.cat([p[name] for p in parts], 1 if name in ("lse", "s_abs") else 0)
            want.setdefault(name, []).append(total)
    want = {name: torch.cat(t, 1 if name in ("lse", "s_abs") else 0) for name, t in want.items()}
    check_forward(o, lse, want, dim)
    for got, name in zip(grads, ("dq", "dk", "dv")):
        within(got, want[name], want[name + "_abs"] + U * want[name].abs() + 1e-6)
