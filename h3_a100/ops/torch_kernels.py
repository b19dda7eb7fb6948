"""PyTorch implementation of the kernel set.

Two jobs: it is the fp32 CPU oracle every CUDA kernel is tested against, and,
with ``kernels.backend: torch`` on a GPU, it is the reference-equivalent
library path (cuBLAS GEMMs, SDPA attention) that the hand-written sm_100a
kernels are measured against.  Every function computes in fp32 and returns
the dtype of its main input unless stated otherwise.

Conventions shared with the native kernels (``h3_a100/ops/native.py``):

* hidden states are 2-D ``[T, H]`` (batch 1 per rank, as in the matched
  contract);
* a modulation row is chosen per token: tokens ``< split`` use row 0, the rest
  row 1 (video+text tokens come first, audio tokens last);
* LoRA for a linear with S output sections (the fused QKV has 3) is stored as
  ``A_cat [S*r, in]`` and ``B_cat [out, r]``; section ``s`` of the output uses
  rows ``s*r:(s+1)*r`` of ``A_cat`` and its own rows of ``B_cat``.  The LoRA
  scale ``s = alpha/r`` is applied exactly once, in ``lora_down``
  (``U = s * x A^T``) and in ``lora_dyb`` (``dyb = s * dy B``); every other
  LoRA term uses those scaled tensors;
* packed batches (``PackedPlan``) keep heads apart: ``[tokens, heads, head_dim]``
  for q and o, ``[tokens, kv_heads, head_dim]`` for k and v, any token and head
  strides (views of a fused projection are fine);
* RoPE rotates interleaved pairs ``(2i, 2i+1)`` of every head with per-token
  tables ``cos, sin: [T, head_dim/2]`` (fp32).
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from .packing import AxisRope, PackedPlan

GELU_C = math.sqrt(2.0 / math.pi)


@dataclass
class Rope:
    cos: torch.Tensor
    sin: torch.Tensor
    head_dim: int
    section_width: int  # columns per output section (hidden size H)
    sections: tuple[int, ...] = (0, 1)  # output sections rotated (q and k)


@dataclass
class GatedResidual:
    residual: torch.Tensor
    gate: torch.Tensor  # [R, H]
    split: int


def _rows(t: int, split: int, table: torch.Tensor) -> torch.Tensor:
    """Expand a [R, H] table to [T, H] by the split rule (fp32)."""
    table = table.float()
    if table.shape[0] == 1 or split >= t:
        return table[0].expand(t, -1)
    if split <= 0:
        return table[1].expand(t, -1)
    return torch.cat([table[0].expand(split, -1), table[1].expand(t - split, -1)], 0)


def gelu_tanh(x: torch.Tensor) -> torch.Tensor:
    return 0.5 * x * (1.0 + torch.tanh(GELU_C * (x + 0.044715 * x * x * x)))


def gelu_tanh_grad(x: torch.Tensor) -> torch.Tensor:
    inner = GELU_C * (x + 0.044715 * x * x * x)
    th = torch.tanh(inner)
    return 0.5 * (1.0 + th) + 0.5 * x * (1.0 - th * th) * GELU_C * (1.0 + 3 * 0.044715 * x * x)


def rope_apply(y: torch.Tensor, rope: Rope, inverse: bool = False) -> torch.Tensor:
    """Rotate the selected sections of ``y [T, S*H]`` (returns a new fp32 tensor)."""
    t = y.shape[0]
    out = y.float().clone()
    sec_width = rope.section_width
    cos = rope.cos.float()[:, None, :]
    sin = rope.sin.float()[:, None, :]
    if inverse:
        sin = -sin
    for s in rope.sections:
        part = out[:, s * sec_width:(s + 1) * sec_width].view(t, -1, rope.head_dim // 2, 2)
        even, odd = part[..., 0].clone(), part[..., 1].clone()
        part[..., 0] = even * cos - odd * sin
        part[..., 1] = even * sin + odd * cos
    return out


class TorchKernels:
    name = "torch"
    native = False

    # ---------------- norm + AdaLN modulate ----------------
    def norm_modulate(self, x, shift, scale, split, eps=1e-6):
        xf = x.float()
        r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
        y = xf * r * (1.0 + _rows(x.shape[0], split, scale)) + _rows(x.shape[0], split, shift)
        return y.to(x.dtype)

    def norm_modulate_bwd(self, x, dy, scale, split, eps=1e-6, add=None, gate=None):
        """dx = add + d(norm_modulate)/dx^T dy; with ``gate`` also returns gate[row] * dx."""
        xf, g = x.float(), dy.float() * (1.0 + _rows(x.shape[0], split, scale))
        r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
        n = xf * r
        dx = r * (g - n * (g * n).mean(-1, keepdim=True))
        if add is not None:
            dx = dx + add.float()
        dx = dx.to(x.dtype)
        if gate is None:
            return dx
        return dx, (dx.float() * _rows(x.shape[0], split, gate)).to(x.dtype)

    # ---------------- linear layers with LoRA ----------------
    def lora_down(self, x, a_cat, scale=1.0):
        return (scale * (x.float() @ a_cat.float().t())).to(x.dtype)

    def _lora_up(self, y, u, b_cat, sections):
        n = y.shape[1]
        r = u.shape[1] // sections
        width = n // sections
        for s in range(sections):
            y[:, s * width:(s + 1) * width] += (
                u[:, s * r:(s + 1) * r].float() @ b_cat[s * width:(s + 1) * width].float().t()
            )
        return y

    def linear(self, x, w, b=None, u=None, b_cat=None, sections=1, epilogue=None):
        """y = x w^T + b (+ U B^T, the LoRA up-projection) then the epilogue.

        epilogue: None | "gelu" (returns (pre, post)) | Rope | GatedResidual.
        """
        if x.dtype == torch.float32:
            y = x @ w.t()
            if b is not None:
                y = y + b
        else:
            y = (torch.addmm(b, x, w.t()) if b is not None else x @ w.t()).float()
        if u is not None:
            y = self._lora_up(y, u, b_cat, sections)
        if epilogue is None:
            return y.to(x.dtype)
        if epilogue == "gelu":
            pre = y.to(x.dtype)
            return pre, gelu_tanh(pre.float()).to(x.dtype)
        if isinstance(epilogue, Rope):
            return rope_apply(y.to(x.dtype), epilogue).to(x.dtype)
        if isinstance(epilogue, GatedResidual):
            gate = _rows(x.shape[0], epilogue.split, epilogue.gate)
            return (epilogue.residual.float() + gate * y.to(x.dtype).float()).to(x.dtype)
        raise ValueError(f"unknown epilogue {epilogue!r}")

    def lora_dyb(self, dy, b_cat, sections, scale=1.0):
        n = dy.shape[1]
        width = n // sections
        parts = [dy[:, s * width:(s + 1) * width].float() @ b_cat[s * width:(s + 1) * width].float()
                 for s in range(sections)]
        return (scale * torch.cat(parts, 1)).to(dy.dtype)

    def linear_dx(self, dy, w, dyb=None, a_cat=None, gelu_pre=None):
        """dx = dy w + dyb A_cat; with ``gelu_pre`` also applies the GELU derivative."""
        if dy.dtype == torch.float32:
            dx = dy @ w
        else:
            dx = (dy @ w).float()
        if dyb is not None:
            dx = dx + dyb.float() @ a_cat.float()
        dx = dx.to(dy.dtype)
        if gelu_pre is not None:
            dx = self.gelu_bwd(dx, gelu_pre)
        return dx

    def lora_wgrad(self, dy, x, u, dyb, sections, grad_a, grad_b):
        """Accumulate dA_cat = dyb^T x and dB_s = dy_s^T U_s into the fp32 sinks."""
        grad_a += dyb.float().t() @ x.float()
        n = dy.shape[1]
        width = n // sections
        r = u.shape[1] // sections
        for s in range(sections):
            grad_b[s * width:(s + 1) * width] += (
                dy[:, s * width:(s + 1) * width].float().t() @ u[:, s * r:(s + 1) * r].float()
            )

    # ---------------- elementwise helpers ----------------
    def gelu_bwd(self, dy, pre):
        return (dy.float() * gelu_tanh_grad(pre.float())).to(dy.dtype)

    def gate_mul(self, dout, gate, split):
        return (dout.float() * _rows(dout.shape[0], split, gate)).to(dout.dtype)

    def rope_bwd(self, dqkv, rope: Rope):
        return rope_apply(dqkv, rope, inverse=True).to(dqkv.dtype)

    # ---------------- attention ----------------
    @staticmethod
    def _split_heads(qkv, heads, head_dim):
        t = qkv.shape[0]
        q, k, v = qkv.view(t, 3, heads, head_dim).permute(1, 2, 0, 3).unbind(0)
        return q, k, v

    def attention_fwd(self, qkv, heads, head_dim):
        q, k, v = self._split_heads(qkv, heads, head_dim)
        if qkv.dtype == torch.float32:
            s = (q @ k.transpose(-1, -2)) / math.sqrt(head_dim)
            lse = torch.logsumexp(s, -1)
            o = torch.softmax(s, -1) @ v
        else:
            o = F.scaled_dot_product_attention(q[None], k[None], v[None])[0]
            lse = None
        return o.transpose(0, 1).reshape(qkv.shape[0], heads * head_dim), lse

    def attention_bwd(self, qkv, o, lse, do, heads, head_dim):
        with torch.enable_grad():
            qkv_ = qkv.detach().requires_grad_(True)
            q, k, v = self._split_heads(qkv_, heads, head_dim)
            if qkv.dtype == torch.float32:
                p = torch.softmax((q @ k.transpose(-1, -2)) / math.sqrt(head_dim), -1)
                out = p @ v
            else:
                out = F.scaled_dot_product_attention(q[None], k[None], v[None])[0]
            out = out.transpose(0, 1).reshape(qkv.shape[0], heads * head_dim)
            (dqkv,) = torch.autograd.grad(out, qkv_, do)
        return dqkv

    # ---------------- packed sequences ----------------
    @staticmethod
    def _axis_tables(rope: AxisRope | None, head_dim: int, x: torch.Tensor):
        """cos, sin [T, 1, head_dim / 2]; pairs without an axis do not turn."""
        half = head_dim // 2
        angles = torch.zeros(x.shape[0], half, dtype=torch.float64, device=x.device)
        if rope is not None:
            if rope.positions.shape[0] != x.shape[0] or sum(rope.pairs) > half:
                raise ValueError("the rotation does not fit q's tokens and head_dim")
            n = sum(rope.pairs)
            angles[:, :n] = rope.positions.double()[:, rope.axis_of_pairs()] * rope.freqs.double()
        dtype = torch.promote_types(x.dtype, torch.float32)
        return angles.cos().to(dtype)[:, None], angles.sin().to(dtype)[:, None]

    @staticmethod
    def _turn(x, cos, sin, interleaved: bool):
        a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
        y = a * cos - b * sin, a * sin + b * cos
        return torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)

    def rope_axes(self, q, k, rope: AxisRope | None, inverse: bool = False):
        """Rotate every head of ``q`` and ``k`` (``k`` may be None); ``inverse`` turns gradients back.

        Without a ``rope`` nothing turns and the results are copies.
        """
        cos, sin = self._axis_tables(rope, q.shape[-1], q)
        sin, interleaved = -sin if inverse else sin, rope is None or rope.interleaved
        return tuple(None if x is None else self._turn(x.to(cos.dtype), cos, sin, interleaved).to(x.dtype)
                     for x in (q, k))

    def qk_norm_rope(self, q, k, q_weight, k_weight, rope: AxisRope | None = None, eps=1e-6):
        """RMS norm of every head of ``q`` and ``k`` (weights ``[head_dim]``), then the rotation."""
        cos, sin = self._axis_tables(rope, q.shape[-1], q)
        out = []
        for x, w in ((q, q_weight), (k, k_weight)):
            xf = x.to(cos.dtype)
            n = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.to(cos.dtype)
            out.append(self._turn(n, cos, sin, rope is None or rope.interleaved).to(x.dtype))
        return tuple(out)

    def qk_norm_rope_bwd(self, q, k, q_weight, k_weight, rope: AxisRope | None, dq, dk, eps=1e-6, out=None):
        """Gradients ``(dq, dk, dq_weight, dk_weight)`` from those of the outputs; the weights' in fp32.

        ``out``: two tensors (views are fine, not over the inputs) to write dq and dk into.
        """
        cos, sin = self._axis_tables(rope, q.shape[-1], q)
        grads, weights = [], []
        for x, w, dy in ((q, q_weight, dq), (k, k_weight, dk)):
            xf = x.to(cos.dtype)
            r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
            n = xf * r
            g = self._turn(dy.to(cos.dtype), cos, -sin, rope is None or rope.interleaved)
            gw = g * w.to(cos.dtype)
            grads.append((r * (gw - n * (gw * n).mean(-1, keepdim=True))).to(x.dtype))
            weights.append((g * n).sum((0, 1)))
        if out is not None:
            grads = [o.copy_(g) for o, g in zip(out, grads)]
        return grads[0], grads[1], weights[0], weights[1]

    def packed_plan(self, q_lens, k_lens=None, *, heads, kv_heads, head_dim, causal=False) -> PackedPlan:
        return PackedPlan.lengths(q_lens, k_lens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, causal=causal)

    @staticmethod
    def _check_packed(q, k, v, plan: PackedPlan) -> None:
        want_q = (plan.q_tokens, plan.heads, plan.head_dim)
        want_k = (plan.k_tokens, plan.kv_heads, plan.head_dim)
        if tuple(q.shape) != want_q or tuple(k.shape) != want_k or tuple(v.shape) != want_k:
            raise ValueError(f"q, k, v must be {want_q}, {want_k}, {want_k} as planned, got "
                             f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")

    @staticmethod
    def _packed_sequences(plan: PackedPlan, device):
        """(query rows, key rows, hidden mask or None) of every sequence."""
        q0 = k0 = 0
        for nq, nk in zip(plan.q_lens, plan.k_lens):
            hidden = None
            if plan.causal:
                i, j = torch.arange(nq, device=device), torch.arange(nk, device=device)
                hidden = j[None, :] - nk > i[:, None] - nq
            yield slice(q0, q0 + nq), slice(k0, k0 + nk), hidden
            q0, k0 = q0 + nq, k0 + nk

    def attention_packed_fwd(self, q, k, v, plan: PackedPlan, scale=None):
        """Attention of each sequence of a packed batch with itself -> (o, lse [heads, tokens] fp32).

        ``q [tokens, heads, D]``, ``k, v [tokens, kv_heads, D]``; query head ``h``
        reads key head ``h // (heads // kv_heads)``.  ``scale`` defaults to
        ``1 / sqrt(D)``.  A query that sees no key gives o = 0 and lse = -inf.
        Values of keys that a query does not see have no weight, but as in any
        product 0 * NaN is NaN: keys and values within one sequence must be finite.
        What lies outside a sequence (other sequences of the batch) is never read into it.
        """
        self._check_packed(q, k, v, plan)
        scale = plan.head_dim ** -0.5 if scale is None else scale
        group = plan.heads // plan.kv_heads
        dtype = torch.promote_types(q.dtype, torch.float32)
        o = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.full((plan.heads, q.shape[0]), -math.inf, dtype=dtype, device=q.device)
        for rq, rk, hidden in self._packed_sequences(plan, q.device):
            if rq.start == rq.stop or rk.start == rk.stop:
                continue
            qs = q[rq].to(dtype).transpose(0, 1)
            ks, vs = (x[rk].to(dtype).transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
            s = scale * (qs @ ks.transpose(1, 2))
            if hidden is not None:
                s = s.masked_fill(hidden, -math.inf)
            row = torch.logsumexp(s, -1)
            p = torch.exp(s - row.masked_fill(row == -math.inf, 0.0)[..., None])
            o[rq] = (p @ vs).transpose(0, 1).to(o.dtype)
            lse[:, rq] = row
        return o, lse

    def attention_packed_bwd(self, q, k, v, o, lse, do, plan: PackedPlan, scale=None, out=None):
        """Gradients ``(dq, dk, dv)``; ``out``: three tensors (views are fine) to write them into."""
        self._check_packed(q, k, v, plan)
        scale = plan.head_dim ** -0.5 if scale is None else scale
        group = plan.heads // plan.kv_heads
        dtype = torch.promote_types(q.dtype, torch.float32)
        if out is not None and len(out) != 3:
            raise ValueError("out must hold dq, dk and dv")
        grads = tuple(torch.zeros(x.shape, dtype=x.dtype, device=x.device) for x in out or (q, k, v))
        for rq, rk, hidden in self._packed_sequences(plan, q.device):
            if rq.start == rq.stop or rk.start == rk.stop:
                continue
            qs, dos, os_ = (x[rq].to(dtype).transpose(0, 1) for x in (q, do, o))
            ks, vs = (x[rk].to(dtype).transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
            s = scale * (qs @ ks.transpose(1, 2))
            row = lse[:, rq].to(dtype)
            p = torch.exp(s - row.masked_fill(row == -math.inf, math.inf)[..., None])
            if hidden is not None:
                p = p.masked_fill(hidden, 0.0)
            ds = scale * p * (dos @ vs.transpose(1, 2) - (dos * os_).sum(-1, keepdim=True))

            def per_key_head(x):
                return x.unflatten(0, (plan.kv_heads, group)).sum(1).transpose(0, 1)

            grads[0][rq] = (ds @ ks).transpose(0, 1).to(grads[0].dtype)
            grads[1][rk] = per_key_head(ds.transpose(1, 2) @ qs).to(grads[1].dtype)
            grads[2][rk] = per_key_head(p.transpose(1, 2) @ dos).to(grads[2].dtype)
        return grads if out is None else tuple(o.copy_(g) for o, g in zip(out, grads))

    # ---------------- small projections ----------------
    def adaln_project(self, temb, w, b):
        """SiLU(temb) @ w^T + b in fp32; temb [R, D_t], w [6H, D_t] -> [R, 6H]."""
        return F.silu(temb.float()) @ w.float().t() + b.float()

    # ---------------- optimizer ----------------
    def sum_squares(self, t):
        return t.float().pow(2).sum().reshape(1)

    def adamw_step(self, master, exp_avg, exp_avg_sq, grad, param_out, norm, *, lr, beta1, beta2, eps,
                   weight_decay, step, max_norm):
        g = grad.float()
        if max_norm and max_norm > 0:
            g = g * torch.clamp(max_norm / (norm.float() + 1e-6), max=1.0)
        master.mul_(1.0 - lr * weight_decay)
        exp_avg.mul_(beta1).add_(g, alpha=1.0 - beta1)
        exp_avg_sq.mul_(beta2).addcmul_(g, g, value=1.0 - beta2)
        bc1, bc2 = 1.0 - beta1 ** step, 1.0 - beta2 ** step
        denom = (exp_avg_sq.sqrt() / math.sqrt(bc2)).add_(eps)
        master.addcdiv_(exp_avg, denom, value=-lr / bc1)
        param_out.copy_(master[:param_out.numel()])

    # ---------------- DMD / flow elementwise ----------------
    def flow_step(self, xt, velocity, sigma, sigma_next, out_dtype):
        """(x0 = xt + sigma*v, xt' = xt + (sigma - sigma')*v) in one pass; x0 in fp32."""
        x0 = xt.float() + sigma * velocity.float()
        nxt = (xt.float() + (sigma - sigma_next) * velocity.float()).to(out_dtype)
        return x0, nxt

    def x0_from_velocity(self, xt, velocity, sigma):
        return xt.float() + sigma * velocity.float()

    def add_noise(self, x0, noise, sigma):
        return ((1.0 - sigma) * x0.float() + sigma * noise.float()).to(x0.dtype)

    def randn(self, shape, dtype, device, generator=None):
        return torch.randn(shape, dtype=dtype, device=device, generator=generator)

    def dmd_loss(self, generated, x0_fake, x0_real):
        from ..trainer.dmd_math import dmd_loss
        return dmd_loss(generated, x0_fake, x0_real)

    def mse_loss(self, pred, target):
        return torch.mean((pred.float() - target.float()) ** 2)
