"""Measured cases of the packed-sequence operators.

Three operators of the kernel set, each in its plain form (elementary torch
operations in fp32) and through the framework's entry points:

* ``rope_axes``         rotary positions with several axes (time, height, width);
* ``qk_norm_rope``      RMS norm of every query and key head with that rotation
                        in the same pass, and its gradients;
* ``attention_packed``  attention over packed sequences of different lengths,
                        causal or not, with grouped heads, and its gradients.

``run`` makes one call of one operator, forward alone or forward and backward
(``train``).
"""

import math

import torch

own = False

EPS = 1e-6
BASE = 10000.0
# The largest fp32 score tensor of a plain form: elements of [sequences, heads, longest, longest].
MAX_SCORES = 6_000_000_000
MAX_SCORES_TRAIN = 3_400_000_000


def listed():
    return [
        # A prompt of 77 tokens rotated alone, at the toy model's 4 heads of 64: the smallest call.
        dict(name="rope_text_77", op="rope", grid="0x0x0", text=77, heads=4, kv_heads=4, head_dim=64,
             dtype="bf16", interleaved=True),
        # Queries and keys of a joint video, text and audio sequence: 31 x 24 x 42 patches, 512 and 5,970 tokens,
        # 42 heads of 128.
        dict(name="rope_video_37730", op="rope", grid="31x24x42", text=512 + 5970, heads=42, kv_heads=42,
             head_dim=128, dtype="bf16", interleaved=True),
        # The next token of five sequences, grouped heads: a latency-bound call of a generating model.
        dict(name="norm_rope_5_tokens", op="norm_rope", train=False, grid="0x0x0", text=5, heads=32, kv_heads=8,
             head_dim=128, dtype="bf16", interleaved=False),
        # The attention input of one joint block at full length: 37,730 tokens, 42 heads of 128.
        dict(name="norm_rope_video_37730", op="norm_rope", train=False, grid="31x24x42", text=512 + 5970, heads=42,
             kv_heads=42, head_dim=128, dtype="bf16", interleaved=True),
        # A training step over a packed batch of an odd length with grouped heads.
        dict(name="norm_rope_train_16411", op="norm_rope", train=True, grid="21x24x31", text=787, heads=32,
             kv_heads=8, head_dim=128, dtype="bf16", interleaved=True),
        # The toy model's heads in fp32, pairs split by halves, forward and backward.
        dict(name="norm_rope_train_f32", op="norm_rope", train=True, grid="16x16x19", text=137, heads=4, kv_heads=4,
             head_dim=64, dtype="f32", interleaved=False),
        # Eight prompts of a text encoder, one of a single token: short causal sequences, grouped heads.
        dict(name="attn_prompts", op="attn", train=False, q_lens="77,1,512,33,128,205,16,301", k_lens="same",
             heads=32, kv_heads=8, head_dim=128, causal=True),
        # One new token for each of twelve sequences over keys of very different lengths.
        dict(name="attn_one_token", op="attn", train=False, q_lens="1,1,1,1,1,1,1,1,1,1,1,1",
             k_lens="32768,777,12001,1,8192,20480,129,30011,4096,16385,64,26000", heads=32, kv_heads=8,
             head_dim=128, causal=True),
        # Three clips of different resolution in one bidirectional call (31 x 12 x 21 patches and less, with text).
        dict(name="attn_clips", op="attn", train=False, q_lens="8324,4109,2523", k_lens="same", heads=16, kv_heads=16,
             head_dim=128, causal=False),
        # The full joint sequence under a causal mask, four of its heads (one rank of a head-parallel run).
        dict(name="attn_video_causal", op="attn", train=False, q_lens="37730", k_lens="same", heads=4, kv_heads=4,
             head_dim=128, causal=True),
        # A training step over clips with grouped heads, causal, one short and one single-token sequence among them.
        dict(name="attn_train_clips", op="attn", train=True, q_lens="8324,4109,131,1", k_lens="same", heads=12,
             kv_heads=4, head_dim=128, causal=True),
        # The toy model's heads: ragged bidirectional captions, forward and backward.
        dict(name="attn_train_d64", op="attn", train=True, q_lens="1040,333,64,900,2,511", k_lens="same", heads=4,
             kv_heads=4, head_dim=64, causal=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rope", "norm_rope", "norm_rope", "attn", "attn", "attn"])
    if op != "attn":
        kv_heads = rng.choice([1, 2, 4, 6, 8, 14])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
        tokens = _log_int(rng, 1, 37_000)
        grid = [0, 0, 0]
        if tokens > 64 and rng.random() < 0.75:
            grid = [_log_int(rng, 1, 31), 0, 0]
            grid[1] = _log_int(rng, 1, min(48, max(1, tokens // grid[0])))
            grid[2] = max(1, min(84, tokens // (grid[0] * grid[1])))
        text = max(1, min(6000, tokens - grid[0] * grid[1] * grid[2]))
        case = dict(op=op, grid="x".join(map(str, grid)), text=text, heads=heads, kv_heads=kv_heads,
                    head_dim=rng.choice([64, 128]), dtype=rng.choice(["bf16", "bf16", "f32"]), interleaved=rng.random() < 0.5)
        if op == "norm_rope":
            case["train"] = rng.random() < 0.5
        return case
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7])
    case = dict(op=op, train=False, heads=heads, kv_heads=kv_heads, head_dim=rng.choice([64, 128]),
                causal=rng.random() < 0.6)
    if rng.random() < 0.25:                      # a few new tokens over long keys
        count = rng.randint(1, 16)
        case["q_lens"] = ",".join(str(rng.choice([1, 1, 1, 2, 5])) for _ in range(count))
        case["k_lens"] = ",".join(str(_log_int(rng, 5, 32768)) for _ in range(count))
        return case
    case["train"] = rng.random() < 0.5
    most = MAX_SCORES_TRAIN if case["train"] else MAX_SCORES
    count = rng.randint(1, 8)
    longest = int(math.sqrt(most / 2 / (count * heads)))
    first = _log_int(rng, 16, min(20_000, longest))
    case["q_lens"] = ",".join(map(str, [first] + [_log_int(rng, 1, first) for _ in range(count - 1)]))
    case["k_lens"] = "same"
    return case


def _axis_pairs(head_dim, grid):
    """Rotation pairs of the three axes; a text-only call rotates by its first axis alone."""
    pairs = head_dim // 2
    if grid[0] == 0:
        return (pairs, 0, 0)
    t = pairs // 4
    h = (pairs - t) // 2
    return (t, h, pairs - t - h)


def _lens(case):
    q_lens = [int(n) for n in case["q_lens"].split(",")]
    return q_lens, q_lens if case["k_lens"] == "same" else [int(n) for n in case["k_lens"].split(",")]


def _grid(case):
    return tuple(int(n) for n in case["grid"].split("x"))


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(shape, generator=gen, device=device, dtype=torch.float32).to(dtype)

    state = {"case": case}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "attn":
        q_lens, k_lens = _lens(case)
        tq, tk = sum(q_lens), sum(k_lens)
        if case["k_lens"] == "same":
            # views of one fused projection, as a block has them
            qkv = normal(tq, (heads + 2 * kv_heads) * dim)
            q = qkv[:, :heads * dim].view(tq, heads, dim)
            k = qkv[:, heads * dim:(heads + kv_heads) * dim].view(tq, kv_heads, dim)
            v = qkv[:, (heads + kv_heads) * dim:].view(tq, kv_heads, dim)
        else:
            q, k, v = normal(tq, heads, dim), normal(tk, kv_heads, dim), normal(tk, kv_heads, dim)
        state.update(q=q, k=k, v=v)
        if case["train"]:
            state["do"] = normal(tq, heads, dim)
        state["cu_q"] = torch.tensor([0] + q_lens, device=device).cumsum(0)
        state["cu_k"] = torch.tensor([0] + k_lens, device=device).cumsum(0)
        if own:
            from h3_a100.ops import get_kernels

            state["kernels"] = get_kernels("native", device)
            state["plan"] = state["kernels"].packed_plan(q_lens, k_lens, heads=heads, kv_heads=kv_heads, head_dim=dim,
                                                         causal=case["causal"])
        return state
    dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    frames, height, width = _grid(case)
    n_text, n_video = case["text"], frames * height * width
    tokens = n_video + n_text
    qkv = normal(tokens, (heads + 2 * kv_heads) * dim, dtype=dtype)
    state["q"] = qkv[:, :heads * dim].view(tokens, heads, dim)
    state["k"] = qkv[:, heads * dim:(heads + kv_heads) * dim].view(tokens, kv_heads, dim)
    # video tokens at their patch's (frame, row, column); other tokens at fractional times of the first axis
    pos = torch.zeros(tokens, 3, device=device)
    if n_video:
        mesh = torch.meshgrid(torch.arange(frames, device=device), torch.arange(height, device=device),
                              torch.arange(width, device=device), indexing="ij")
        pos[:n_video] = torch.stack([m.reshape(-1) for m in mesh], -1).float()
        pos[n_video:, 0] = torch.arange(n_text, device=device).float() * (frames / n_text)
    else:
        pos[:, 0] = torch.arange(n_text, device=device).float() * (min(n_text, 100) / n_text)
    pairs = _axis_pairs(dim, (frames, height, width))
    freqs = torch.cat([BASE ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in pairs]).float().to(device)
    axis = torch.tensor([a for a, n in enumerate(pairs) for _ in range(n)], device=device)   # the axis of each pair
    state.update(positions=pos, freqs=freqs, pairs=pairs, axis=axis)
    if case["op"] == "norm_rope":
        wdtype = torch.float32 if case["train"] else dtype
        state["q_weight"] = (1.0 + 0.2 * normal(dim, dtype=torch.float32)).to(wdtype)
        state["k_weight"] = (1.0 + 0.2 * normal(dim, dtype=torch.float32)).to(wdtype)
        if case["train"]:
            state["dq"] = normal(tokens, heads, dim, dtype=dtype)
            state["dk"] = normal(tokens, kv_heads, dim, dtype=dtype)
    if own:
        from h3_a100.ops import AxisRope, get_kernels

        state["kernels"] = get_kernels("native", device)
        state["rope"] = AxisRope(pos, freqs, pairs, interleaved=case["interleaved"])
    return state


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "rope":
        cos, sin = _tables(state)
        return _rotate(state["q"], cos, sin, case["interleaved"]).to(state["q"].dtype), \
            _rotate(state["k"], cos, sin, case["interleaved"]).to(state["k"].dtype)
    if case["op"] == "norm_rope":
        return _plain_norm_rope(state, case)
    return _plain_attention(state, case)


def _run_own(state, case):
    kernels, q, k = state["kernels"], state["q"], state["k"]
    if case["op"] == "rope":
        return kernels.rope_axes(q, k, state["rope"])
    if case["op"] == "norm_rope":
        out = kernels.qk_norm_rope(q, k, state["q_weight"], state["k_weight"], state["rope"], eps=EPS)
        if not case["train"]:
            return out
        grads = kernels.qk_norm_rope_bwd(q, k, state["q_weight"], state["k_weight"], state["rope"], state["dq"],
                                         state["dk"], eps=EPS)
        return tuple(out) + tuple(grads)
    o, lse = kernels.attention_packed_fwd(q, k, state["v"], state["plan"])
    if not case["train"]:
        return o, lse
    return (o,) + tuple(kernels.attention_packed_bwd(q, k, state["v"], o, lse, state["do"], state["plan"]))


# ---------------------------------------------------------------- plain forms
def _tables(state):
    angles = state["positions"][:, state["axis"]] * state["freqs"]
    return angles.cos()[:, None, :], angles.sin()[:, None, :]


def _halves(x, interleaved):
    if interleaved:
        return x[..., 0::2], x[..., 1::2]
    return x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]


def _join(a, b, interleaved):
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def _rotate(x, cos, sin, interleaved):
    a, b = _halves(x.float(), interleaved)
    return _join(a * cos - b * sin, a * sin + b * cos, interleaved)


def _norm_rotate(x, weight, cos, sin, interleaved):
    x = x.float()
    n = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))
    return _rotate(n * weight.float(), cos, sin, interleaved)


def _norm_rotate_grads(x, weight, dy, cos, sin, interleaved):
    x = x.float()
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * r
    g = _rotate(dy, cos, -sin, interleaved)
    gw = g * weight.float()
    return r * (gw - n * (gw * n).mean(-1, keepdim=True)), (g * n).sum((0, 1))


def _plain_norm_rope(state, case):
    cos, sin = _tables(state)
    q, k, qw, kw, inter = state["q"], state["k"], state["q_weight"], state["k_weight"], case["interleaved"]
    out = (_norm_rotate(q, qw, cos, sin, inter).to(q.dtype), _norm_rotate(k, kw, cos, sin, inter).to(k.dtype))
    if not case["train"]:
        return out
    dq, dqw = _norm_rotate_grads(q, qw, state["dq"], cos, sin, inter)
    dk, dkw = _norm_rotate_grads(k, kw, state["dk"], cos, sin, inter)
    return out + (dq.to(q.dtype), dk.to(k.dtype), dqw, dkw)


def _pad(x, cu, longest):
    """[tokens, heads, dim] -> fp32 [sequences, heads, longest, dim]; rows past a sequence hold some other row."""
    index = (cu[:-1, None] + torch.arange(longest, device=cu.device)).clamp_(max=x.shape[0] - 1)
    return x[index].transpose(1, 2).float()


def _unpad(x, cu, tokens):
    """[sequences, heads, longest, ...] -> [tokens, heads, ...]"""
    t = torch.arange(tokens, device=cu.device)
    seq = torch.searchsorted(cu, t, right=True) - 1
    return x.transpose(1, 2)[seq, t - cu[seq]]


def _plain_attention(state, case):
    q_lens, k_lens = _lens(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    group, count, lq, lk = heads // kv_heads, len(q_lens), max(q_lens), max(k_lens)
    cu_q, cu_k = state["cu_q"], state["cu_k"]
    scale = dim ** -0.5
    # the heads of a group sit in the rows, so that shared keys are not repeated
    q = _pad(state["q"], cu_q, lq).reshape(count, kv_heads, group * lq, dim)
    k, v = _pad(state["k"], cu_k, lk), _pad(state["v"], cu_k, lk)
    nq, nk = (cu_q[1:] - cu_q[:-1])[:, None, None], (cu_k[1:] - cu_k[:-1])[:, None, None]
    row, col = torch.arange(lq, device=cu_q.device)[:, None], torch.arange(lk, device=cu_q.device)[None, :]
    hidden = (col >= nk) | (row >= nq)
    if case["causal"]:
        hidden = hidden | (col - nk > row - nq)
    hidden = hidden[:, None, None]
    s = (q @ k.transpose(-1, -2)).mul_(scale).view(count, kv_heads, group, lq, lk)
    s.masked_fill_(hidden, -math.inf)
    # rows past a sequence are hidden throughout; any finite maximum keeps them free of NaN
    m = s.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = s.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    lse = (m + l.log()).view(count, heads, lq)
    p = p.div_(l.clamp(min=1e-30)).view(count, kv_heads, group * lq, lk)
    o = p @ v
    out = _unpad(o.view(count, heads, lq, dim), cu_q, sum(q_lens))
    if not case["train"]:
        return out.to(torch.bfloat16), _unpad(lse, cu_q, sum(q_lens)).t().contiguous()
    do = _pad(state["do"], cu_q, lq).reshape(count, kv_heads, group * lq, dim)
    dv = p.transpose(-1, -2) @ do
    ds = (do @ v.transpose(-1, -2)).sub_((o * do).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    return (out.to(torch.bfloat16), _unpad(dq.view(count, heads, lq, dim), cu_q, sum(q_lens)).to(torch.bfloat16),
            _unpad(dk, cu_k, sum(k_lens)).to(torch.bfloat16), _unpad(dv, cu_k, sum(k_lens)).to(torch.bfloat16))


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attention(case, state)
    q, k = state["q"].double(), state["k"].double()
    dim, inter = case["head_dim"], case["interleaved"]
    angle = torch.cat([state["positions"][:, a:a + 1].double() * f.double()
                       for a, f in enumerate(state["freqs"].split(list(state["pairs"])))], -1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]      # e^{i angle}

    def rotated(x, turn):
        z = torch.view_as_complex(x.reshape(*x.shape[:-1], dim // 2, 2)) if inter \
            else torch.complex(x[..., :dim // 2], x[..., dim // 2:])
        z = z * turn
        return torch.view_as_real(z).reshape(x.shape) if inter else torch.cat([z.real, z.imag], -1)

    if case["op"] == "rope":
        return rotated(q, turn), rotated(k, turn)

    def normed(x, weight):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight

    qw, kw = state["q_weight"].double(), state["k_weight"].double()
    out = (rotated(normed(q, qw), turn), rotated(normed(k, kw), turn))
    if not case["train"]:
        return out
    grads = []
    for x, w, dy in ((q, qw, state["dq"]), (k, kw, state["dk"])):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        with torch.enable_grad():
            y = normed(x, w)
        grads.append(torch.autograd.grad(y, (x, w), rotated(dy.double(), turn.conj())))
    return out + (grads[0][0], grads[1][0], grads[0][1], grads[1][1])


def _exact_attention(case, state):
    q_lens, k_lens = _lens(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    group, train = heads // kv_heads, case["train"]
    q, k, v = state["q"], state["k"], state["v"]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((heads, q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    dq = torch.zeros_like(o)
    dk = torch.zeros(k.shape, dtype=torch.float64, device=q.device)
    dv = torch.zeros_like(dk)
    q0 = k0 = 0
    for nq, nk in zip(q_lens, k_lens):
        step = max(1, 400_000_000 // max(nk, 1))
        for h in range(heads if nk else 0):
            kh, vh = k[k0:k0 + nk, h // group].double(), v[k0:k0 + nk, h // group].double()
            for i in range(0, nq, step):
                rows = slice(q0 + i, q0 + min(i + step, nq))
                qh = q[rows, h].double()
                s = qh @ kh.T / math.sqrt(dim)
                if case["causal"]:
                    see = torch.arange(nk, device=q.device) <= \
                        torch.arange(i, i + qh.shape[0], device=q.device)[:, None] + (nk - nq)
                    s = torch.where(see, s, -math.inf)
                lse[h, rows] = torch.logsumexp(s, -1)
                p = torch.softmax(s, -1)
                o[rows, h] = p @ vh
                if train:
                    doh = state["do"][rows, h].double()
                    dp = doh @ vh.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(dim)
                    dq[rows, h] = ds @ kh
                    dk[k0:k0 + nk, h // group] += ds.T @ qh
                    dv[k0:k0 + nk, h // group] += p.T @ doh
        q0, k0 = q0 + nq, k0 + nk
    return (o, dq, dk, dv) if train else (o, lse)


# ---------------------------------------------------------------- work
def work(case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "attn":
        q_lens, k_lens = _lens(case)
        if case["causal"]:
            # query i of nq sees nk - nq + i + 1 keys, at least none
            pairs = sum(nq * (2 * nk - nq + 1) // 2 if nk >= nq else nk * (nk + 1) // 2
                        for nq, nk in zip(q_lens, k_lens))
        else:
            pairs = sum(nq * nk for nq, nk in zip(q_lens, k_lens))
        q_bytes, k_bytes = sum(q_lens) * heads * dim * 2, sum(k_lens) * kv_heads * dim * 2
        if not case["train"]:       # q, k, v -> o, lse
            return {"bytes": 2 * q_bytes + 2 * k_bytes + sum(q_lens) * heads * 4, "flops": 4 * dim * heads * pairs}
        # q, k, v, do -> o, dq, dk, dv
        return {"bytes": 4 * q_bytes + 4 * k_bytes, "flops": 14 * dim * heads * pairs}
    frames, height, width = _grid(case)
    tokens = frames * height * width + case["text"]
    size = tokens * (heads + kv_heads) * dim
    elem = 4 if case["dtype"] == "f32" else 2
    tables = tokens * 12 + dim * 2
    if case["op"] == "rope":
        return {"bytes": 2 * size * elem + tables, "flops": 3 * size}
    if not case["train"]:
        return {"bytes": 2 * size * elem + tables + 2 * dim * elem, "flops": 7 * size}
    # q, k, dq, dk -> rotated q, k, their gradients and those of the weights
    return {"bytes": 4 * size * elem + tables + 4 * dim * 4, "flops": 22 * size}
