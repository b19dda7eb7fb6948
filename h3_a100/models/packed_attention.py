"""Self-attention over a packed batch of samples of different lengths.

One layer is: fused QKV projection -> RMS norm of every q and k head with the
rotation by (time, height, width) in the same pass -> attention inside each
sample, causal or not, with grouped key/value heads -> output projection.  The
projections are frozen, as everywhere in this trainer; the norm weights train.
The backward is written out like the DiT block's: the gradient of the fused
projection is assembled in one buffer that the attention and norm kernels write
into directly.

Serving: ``forward`` with ``past`` takes a few new tokens per sample over the
keys and values of the tokens before them (``PackedPlan`` with longer
``k_lens``), the same kernels as for a whole prompt.
"""

from __future__ import annotations

import torch
from torch import nn

from ..ops.packing import AxisRope, PackedPlan


class _PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(fctx, x, q_weight, k_weight, layer, plan, rope):
        K, d = layer.kernels, layer.head_dim
        qkv = K.linear(x, layer.qkv_weight, layer.qkv_bias)
        q, k, v = layer.split(qkv)
        qn, kn = K.qk_norm_rope(q, k, q_weight, k_weight, rope, layer.eps)
        o, lse = K.attention_packed_fwd(qn, kn, v, plan)
        fctx.save_for_backward(qkv, qn, kn, o, lse, q_weight, k_weight)
        fctx.layer, fctx.plan, fctx.rope = layer, plan, rope
        return K.linear(o.view(x.shape[0], layer.heads * d), layer.out_weight, layer.out_bias)

    @staticmethod
    def backward(fctx, dy):
        qkv, qn, kn, o, lse, q_weight, k_weight = fctx.saved_tensors
        layer, rope = fctx.layer, fctx.rope
        K = layer.kernels
        q, k, v = layer.split(qkv)
        do = K.linear_dx(dy.contiguous(), layer.out_weight).view(o.shape)
        dqkv = torch.empty_like(qkv)
        dq, dk, dv = layer.split(dqkv)
        dqn, dkn = torch.empty_like(qn), torch.empty_like(kn)
        K.attention_packed_bwd(qn, kn, v, o, lse, do, fctx.plan, out=(dqn, dkn, dv))
        _, _, dqw, dkw = K.qk_norm_rope_bwd(q, k, q_weight, k_weight, rope, dqn, dkn, layer.eps, out=(dq, dk))
        dx = K.linear_dx(dqkv, layer.qkv_weight) if fctx.needs_input_grad[0] else None
        return dx, dqw.to(q_weight.dtype), dkw.to(k_weight.dtype), None, None, None


class PackedSelfAttention(nn.Module):
    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, kernels, *, eps: float = 1e-6,
                 dtype: torch.dtype = torch.bfloat16, device="cpu") -> None:
        super().__init__()
        if heads % kv_heads:
            raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, head_dim, eps
        object.__setattr__(self, "kernels", kernels)
        width = (heads + 2 * kv_heads) * head_dim

        def frozen(*shape):
            std = shape[-1] ** -0.5 if len(shape) > 1 else 0.0
            return nn.Parameter((torch.randn(*shape, device=device) * std).to(dtype), requires_grad=False)

        self.qkv_weight, self.qkv_bias = frozen(width, hidden), frozen(width)
        self.out_weight, self.out_bias = frozen(hidden, heads * head_dim), frozen(hidden)
        self.q_norm = nn.Parameter(torch.ones(head_dim, device=device))
        self.k_norm = nn.Parameter(torch.ones(head_dim, device=device))

    def split(self, qkv: torch.Tensor):
        """Views ``[tokens, heads, head_dim]`` of q, k and v in a fused ``[tokens, width]`` tensor."""
        h, g, d = self.heads, self.kv_heads, self.head_dim
        t = qkv.shape[0]
        return (qkv[:, :h * d].view(t, h, d), qkv[:, h * d:(h + g) * d].view(t, g, d),
                qkv[:, (h + g) * d:].view(t, g, d))

    def plan(self, q_lens, k_lens=None, *, causal: bool) -> PackedPlan:
        return self.kernels.packed_plan(q_lens, k_lens, heads=self.heads, kv_heads=self.kv_heads,
                                        head_dim=self.head_dim, causal=causal)

    def forward(self, x: torch.Tensor, plan: PackedPlan, rope: AxisRope | None = None, past=None):
        """``x [tokens, hidden]`` of all samples one behind the other -> the same shape.

        With ``past = (keys, values)``, lists with one ``[tokens, kv_heads,
        head_dim]`` tensor per sample, ``x`` holds the new tokens of each sample
        (``plan.k_lens`` counts past and new ones); returns ``(y, (keys,
        values))`` with the new tokens' appended.  No gradient flows then.
        """
        if past is None:
            return _PackedAttentionFn.apply(x, self.q_norm, self.k_norm, self, plan, rope)
        with torch.no_grad():
            K = self.kernels
            q, k, v = self.split(K.linear(x, self.qkv_weight, self.qkv_bias))
            q, k = K.qk_norm_rope(q, k, self.q_norm, self.k_norm, rope, self.eps)
            keys, values = [], []
            for old, new, out in ((past[0], k, keys), (past[1], v, values)):
                for before, now in zip(old, new.split(list(plan.q_lens))):
                    out.append(torch.cat([before, now]))
            o, _ = K.attention_packed_fwd(q, torch.cat(keys), torch.cat(values), plan)
            y = K.linear(o.view(x.shape[0], self.heads * self.head_dim), self.out_weight, self.out_bias)
        return y, (keys, values)
