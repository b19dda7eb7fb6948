"""Descriptions that the packed-sequence operators take: rotation and batch plan.

``AxisRope``    a rotation by positions on several axes (time, height, width);
``PackedPlan``  the lengths of a packed batch and, for the native kernels, its
                work lists on the GPU.

Both are made once per batch layout and used by every layer, forward and backward.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class AxisRope:
    """Rotation of pair ``i`` of every head by ``positions[t, axis(i)] * freqs[i]``.

    ``pairs`` counts the rotation pairs of each axis, in order; pairs past their
    sum (at most ``head_dim / 2``) are left alone.  ``interleaved`` pairs are
    elements ``(2i, 2i + 1)``, as in ``Rope``; otherwise pair ``i`` is elements
    ``(i, i + head_dim / 2)``.  Positions may be fractional.
    """

    positions: torch.Tensor       # [tokens, axes] fp32
    freqs: torch.Tensor           # [sum(pairs)] fp32
    pairs: tuple[int, ...]
    interleaved: bool = True

    def __post_init__(self) -> None:
        self.pairs = tuple(int(n) for n in self.pairs)
        if not 1 <= len(self.pairs) <= 4 or min(self.pairs) < 0:
            raise ValueError(f"a rotation has 1 to 4 axes with a number of pairs each, got {self.pairs}")
        if self.positions.dim() != 2 or self.positions.shape[1] != len(self.pairs):
            raise ValueError(f"positions must be [tokens, {len(self.pairs)}], got {tuple(self.positions.shape)}")
        if self.freqs.shape != (sum(self.pairs),):
            raise ValueError(f"freqs must hold {sum(self.pairs)} values, got {tuple(self.freqs.shape)}")
        if self.positions.dtype != torch.float32 or self.freqs.dtype != torch.float32:
            raise ValueError("positions and freqs must be fp32")

    def axis_of_pairs(self) -> torch.Tensor:
        axes = [a for a, n in enumerate(self.pairs) for _ in range(n)]
        return torch.tensor(axes, dtype=torch.long, device=self.positions.device)


@dataclass(frozen=True)
class PackedPlan:
    """A packed batch: sequences one behind the other on the token axis.

    Sequence ``s`` has ``q_lens[s]`` queries and ``k_lens[s]`` keys (either may
    be zero).  With ``causal``, query ``i`` of ``nq`` sees key ``j`` of ``nk``
    iff ``j - nk <= i - nq``: the last query sees every key, so a few new
    tokens over older keys and a whole prompt are the same call.  Made by
    ``packed_plan`` of a kernel set.
    """

    q_lens: tuple[int, ...]
    k_lens: tuple[int, ...]
    heads: int
    kv_heads: int
    head_dim: int
    causal: bool
    blob: torch.Tensor | None = None      # the native kernels' work lists
    meta: tuple[int, ...] = ()

    @classmethod
    def lengths(cls, q_lens, k_lens, *, heads: int, kv_heads: int, head_dim: int, causal: bool, **native):
        q_lens = tuple(int(n) for n in q_lens)
        k_lens = q_lens if k_lens is None else tuple(int(n) for n in k_lens)
        if len(q_lens) != len(k_lens):
            raise ValueError(f"{len(q_lens)} query lengths but {len(k_lens)} key lengths")
        if min(q_lens + k_lens, default=0) < 0:
            raise ValueError("lengths must not be negative")
        if kv_heads < 1 or heads < 1 or heads % kv_heads:
            raise ValueError(f"heads ({heads}) must be a positive multiple of kv_heads ({kv_heads})")
        return cls(q_lens, k_lens, int(heads), int(kv_heads), int(head_dim), bool(causal), **native)

    @property
    def q_tokens(self) -> int:
        return sum(self.q_lens)

    @property
    def k_tokens(self) -> int:
        return sum(self.k_lens)
