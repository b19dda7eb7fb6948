"""Work lists of packed batches, checked on the CPU.

Every visible (query, key) pair must be in exactly one forward item, one dq
item and one dk/dv item of its key/value head; every query in exactly one
unsplit forward item or one join; no item may reach outside its sequence.
"""

from __future__ import annotations

import random

import pytest
import torch

_C = pytest.importorskip("h3_a100._C")

TQ, TK, HQ, HK, D, FWD, FWD_B, FWD_N, JOIN, JOIN_N, SLOTS, ROWS, DQ, DQ_B, DQ_N, DKV, DKV_B, DKV_N, INTS = range(19)


def _items(ints, at, begin, blocks):
    starts = ints[begin:begin + blocks + 1].tolist()
    assert starts[0] == 0 and starts == sorted(starts)
    return ints[at:at + 8 * starts[-1]].view(-1, 8).tolist(), starts


def _seen(item):
    """[queries, keys] of the item: what each of its queries sees."""
    q0, nq, k0, nk, diag = item[:5]
    i, j = torch.arange(nq)[:, None], torch.arange(nk)[None, :]
    return j <= i + diag


def _expected(q_lens, k_lens, causal):
    want = torch.zeros(sum(q_lens), sum(k_lens), dtype=torch.int32)
    q0 = k0 = 0
    for nq, nk in zip(q_lens, k_lens):
        i, j = torch.arange(nq)[:, None], torch.arange(nk)[None, :]
        want[q0:q0 + nq, k0:k0 + nk] = (j - nk <= i - nq).int() if causal else 1
        q0, k0 = q0 + nq, k0 + nk
    return want


CASES = [
    ([5], None, 1, 1, True), ([128, 1, 0, 77], None, 8, 2, True), ([300, 20], [300, 20], 6, 2, False),
    ([1, 1, 1], [1500, 3, 700], 8, 2, True), ([1], [6000], 4, 4, False), ([9, 200], [4, 100], 3, 3, True),
    ([0, 0], [10, 300], 2, 1, True), ([700], [0], 2, 2, False), ([1300], None, 7, 1, True),
    ([64, 64], None, 256, 2, False),
]


@pytest.mark.parametrize("sms", [1, 13, 148])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,causal", CASES)
def test_every_pair_is_worked_on_once(q_lens, k_lens, heads, kv_heads, causal, sms):
    k_lens = q_lens if k_lens is None else k_lens
    group = heads // kv_heads
    bt = 128 // group
    blob, meta = _C.packed_schedule(q_lens, k_lens, heads, kv_heads, 128, causal, sms)
    assert blob.dtype == torch.int32 and blob.numel() == meta[INTS]
    assert [meta[TQ], meta[TK], meta[HQ], meta[HK], meta[D]] == [sum(q_lens), sum(k_lens), heads, kv_heads, 128]
    ints = blob.clone()
    want = _expected(q_lens, k_lens, causal)
    bounds_q = torch.tensor([0] + q_lens).cumsum(0).tolist()
    bounds_k = torch.tensor([0] + k_lens).cumsum(0).tolist()

    def inside(item):
        q0, nq, k0, nk = item[:4]
        return any(a <= q0 and q0 + nq <= b and c <= k0 and k0 + nk <= d for a, b, c, d in
                   zip(bounds_q, bounds_q[1:], bounds_k, bounds_k[1:]))

    def covered(items):
        got = [torch.zeros_like(want) for _ in range(kv_heads)]
        for item in items:
            assert inside(item)
            q0, nq, k0, nk = item[:4]
            got[item[5]][q0:q0 + nq, k0:k0 + nk] += _seen(item).int()
        return all(torch.equal(g, want) for g in got)

    fwd, starts = _items(ints, meta[FWD], meta[FWD_B], meta[FWD_N])
    assert meta[FWD_N] <= sms and covered(fwd)
    rows = torch.zeros(kv_heads, sum(q_lens), dtype=torch.int32)
    slots = {}
    for item in fwd:
        q0, nq, k0, nk, diag, head, slot, parts = item
        assert nq <= 2 * bt
        if slot < 0:
            rows[head, q0:q0 + nq] += 1
            continue
        for t in range((nq + bt - 1) // bt):
            key = slot + t * parts
            assert key not in slots
            slots[key] = (q0 + t * bt, min(bt, nq - t * bt), head)
        # the second query tile never has fewer key tiles than the first
        seen = _seen(item).any(0)
        assert not seen.any() or nk > 0
    joins = ints[meta[JOIN]:meta[JOIN] + 8 * meta[JOIN_N]].view(-1, 8).tolist()
    for q0, nq, head, slot0, parts, *_ in joins:
        rows[head, q0:q0 + nq] += 1
        assert nq * group <= meta[ROWS]
        for s in range(slot0, slot0 + parts):
            assert slots.pop(s) == (q0, nq, head)
    assert not slots and torch.equal(rows, torch.ones_like(rows))
    assert all(s < meta[SLOTS] for j in joins for s in range(j[3], j[3] + j[4]))

    dq, _ = _items(ints, meta[DQ], meta[DQ_B], meta[DQ_N])
    assert covered(dq) and all(i[1] <= bt for i in dq)
    count = torch.zeros(kv_heads, sum(q_lens), dtype=torch.int32)
    for i in dq:
        count[i[5], i[0]:i[0] + i[1]] += 1
    assert torch.equal(count, torch.ones_like(count))

    dkv, _ = _items(ints, meta[DKV], meta[DKV_B], meta[DKV_N])
    assert covered(dkv) and all(i[3] <= 128 for i in dkv)
    count = torch.zeros(kv_heads, sum(k_lens), dtype=torch.int32)
    for i in dkv:
        count[i[5], i[2]:i[2] + i[3]] += 1
    assert torch.equal(count, torch.ones_like(count))


def test_random_batches():
    rng = random.Random(7)
    for _ in range(40):
        kv = rng.choice([1, 2, 3])
        n = rng.randint(1, 5)
        q = [rng.choice([0, 1, 2, 127, 129, rng.randint(1, 900)]) for _ in range(n)]
        k = q if rng.random() < 0.5 else [rng.choice([0, 1, 128, rng.randint(1, 2500)]) for _ in range(n)]
        test_every_pair_is_worked_on_once(q, k, kv * rng.choice([1, 3, 4, 7]), kv, rng.random() < 0.6,
                                          rng.choice([1, 4, 40]))


def test_long_keys_are_split_and_level():
    """One new token over long keys: every block gets about the same number of key tiles."""
    blob, meta = _C.packed_schedule([1] * 3, [30000, 500, 12000], 32, 8, 128, True, 148)
    assert meta[JOIN_N] > 0 and meta[FWD_N] >= 140
    items, starts = _items(blob, meta[FWD], meta[FWD_B], meta[FWD_N])
    loads = [sum((i[3] + 127) // 128 for i in items[a:b]) for a, b in zip(starts, starts[1:])]
    assert max(loads) <= 1.5 * (sum(loads) / 148) + 4


@pytest.mark.parametrize("args,message", [
    (([1, 2], [1], 4, 4, 128, True, 8), "as many"), (([1], [1], 5, 2, 128, True, 8), "multiple"),
    (([1], [1], 4, 4, 96, True, 8), "head_dim"), (([-1], [1], 4, 4, 64, True, 8), "negative"),
    (([1], [1], 258, 2, 64, True, 8), "128 query heads"), (([1 << 28], [1], 1, 1, 64, False, 8), "2\\^28"),
])
def test_refusals(args, message):
    with pytest.raises(RuntimeError, match=message):
        _C.packed_schedule(*args)
