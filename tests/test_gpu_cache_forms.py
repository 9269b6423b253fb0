"""Every form of the cache operators' kernels against the definitions in 64 bits:
tree workgroups of 32, 64, 128 and 256 rows over several stages of keys, the merge
of many splits, both forms of the eviction's moves and every one of its selection.
FORMS holds the tree calls with the rows of a workgroup and the splits that they are to run with;
test_cache_plans.py holds the library's plan to it."""

from __future__ import annotations

import math
import sys

import pytest
import torch

import cache_ops_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16

# B, Hq, Hkv, capacity, T, lengths, requested splits: rows of a workgroup, splits
FORMS = [
    ((20, 32, 8, 1500, 16, [1500, 0, 1, 16, 1027, 15, 256, 1290, 4000, 17] * 2, 1), (64, 1)),
    ((6, 12, 12, 1900, 130, [1900, 130, 129, 1111, 641, 2000], 2), (64, 2)),
    ((12, 64, 8, 2000, 65, [2000, 1024, 1025, 0, 64, 65, 66, 333, 1999, 1500, 777, 2000], 1), (128, 1)),
    ((8, 24, 8, 1300, 130, [1300, 1299, 130, 0, 131, 700, 513, 1024], 1), (128, 1)),
    ((1, 16, 8, 40000, 128, [39333], 0), (128, 16)),
    ((1, 32, 8, 40000, 64, [39987], 0), (256, 32)),
    ((16, 64, 16, 1700, 130, [1700, 0, 129, 130, 131, 1024, 1280, 1281, 1699, 1500, 600, 1, 257, 900, 1234, 2000], 2),
     (256, 2)),
    # the merge of many splits, some of them a shorter sequence's own
    ((2, 3, 1, 2304, 5, [2304, 700], 9), (32, 9)),
    ((3, 7, 1, 4352, 3, [4352, 4097, 0], 17), (32, 17)),
    ((2, 5, 1, 8448, 5, [8448, 256], 33), (32, 33)),
    ((3, 11, 1, 16640, 1, [16640, 1, 9000], 65), (32, 65)),
    ((1, 16, 1, 40000, 2, [39999], 0), (32, 157)),
]


def _say(label):
    print(f"[gpu case] {label}", file=sys.stderr, flush=True)


def _randn(shape, gen, dtype, dev):
    return torch.randn(shape, generator=gen, device=dev).to(dtype)


def _masks(B, T, seed):
    """Trees of each sequence, their depth not bounded by a word of the packed masks."""
    from SSA import tree_mask_from_parents

    g = torch.Generator().manual_seed(seed)
    back = torch.randint(1, 90, (B, T), generator=g)
    return tree_mask_from_parents((torch.arange(T) - back).clamp_min(-1))


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("call", [c for c, _ in FORMS])
def test_tree_forms(gpu, call, dtype, D):
    from SSA import ssa_tree_attention

    B, Hq, Hk, cap, T, lens, splits = call
    _say(f"tree form D={D} {dtype} {call}")
    g = torch.Generator(device=gpu).manual_seed(D + T)
    k, v = _randn((B, Hk, cap, D), g, dtype, gpu), _randn((B, Hk, cap, D), g, dtype, gpu)
    q = _randn((B, Hq, T, D), g, dtype, gpu)
    mask = _masks(B, T, T).to(gpu)
    if T > 3:
        mask[0, T // 2] = False  # a node without even itself
    scale, n, b = 1.0 / math.sqrt(D), 1.5, 0.8
    lens32 = torch.tensor(lens, dtype=torch.int32, device=gpu)
    scalars = torch.tensor(n, device=gpu), torch.tensor(b, device=gpu)
    out, m = ssa_tree_attention(q, k, v, lens32, mask, scale, *scalars, num_splits=splits, return_m=True)
    torch.cuda.synchronize()
    want, wm, tol, mtol = ref.tree(q, k, v, lens, mask, scale, n, b)
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), f"out: {float((off - tol).max())} over its bound, error {float(off.max())}"
    empty = wm == -math.inf
    assert torch.equal(m == -math.inf, empty)
    moff = torch.where(empty, torch.zeros_like(wm), (m.double() - wm).abs())
    assert bool((moff <= mtol).all()), f"m: {float((moff - mtol).max())} over its bound"
    # NaN and infinities behind the sequences reach nothing
    for i, L in enumerate(lens):
        k[i, :, L:], v[i, :, L:] = math.nan, math.inf
    again, am = ssa_tree_attention(q, k, v, lens32, mask, scale, *scalars, num_splits=splits, return_m=True)
    assert torch.equal(again, out) and torch.equal(am, m)


def _evicted(lens, weights, keep, sinks, recent):
    """(new lengths, weights, kept) by stable sorts: of equal weights the lower row, NaN lowest."""
    B, Hk, cap = weights.shape
    w = weights.double()
    at = torch.arange(cap, device=w.device)
    L = torch.tensor([min(max(x, 0), cap) for x in lens], device=w.device)[:, None, None]
    rank = w.masked_fill(w.isnan(), -math.inf)
    # three levels above each other: rows past the length, NaN, numbers, rows that stay in any case
    level = torch.where(w.isnan(), 1, 2).masked_fill((at < sinks) | (at >= L - recent), 3).masked_fill(at >= L, 0)
    by_weight = rank.masked_fill(level == 3, 0.0).sort(dim=-1, descending=True, stable=True)[1]
    order = by_weight.gather(-1, level.gather(-1, by_weight).sort(dim=-1, descending=True, stable=True)[1])
    new = L.clamp(max=keep)
    whole = L <= keep
    order = torch.where(whole, at.expand_as(order), order)[..., :keep]
    inside = torch.arange(keep, device=w.device) < new
    kept = order.masked_fill(~inside, cap).sort(-1)[0]
    left = torch.zeros_like(weights)
    left[..., :keep] = weights.gather(-1, kept.clamp(max=cap - 1)).masked_fill(~inside, 0.0)
    return new[:, 0, 0], left, kept.masked_fill(~inside, -1).int()


def _odd_weights(B, Hk, cap, seed, dev):
    """Spread weights with ties, zeros, NaN and infinities among them."""
    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randn(B, Hk, cap, generator=g, device=dev).mul_(1.5).exp_()
    pick = torch.rand(B, Hk, cap, generator=g, device=dev)
    w = torch.where(pick < 0.3, (4 * w).round() / 4, w)
    for lo, value in ((0.30, 0.0), (0.32, -0.0), (0.33, math.nan), (0.34, math.inf), (0.345, -1.0)):
        w = torch.where((pick >= lo) & (pick < lo + 0.005), torch.full_like(w, value), w)
    return w


@pytest.mark.parametrize("dtype,layout", [(BF16, "bhsd"), (FP16, "bshd")])
@pytest.mark.parametrize(
    "B,Hk,cap,D,lens,keep,sinks,recent",
    [
        # 48 to 64 heads at head dim 64 and 32 at 128: moves in slices of 64 bytes, several
        # chunks of 1024 rows and a part of one
        (6, 8, 5000, 64, [5000, 4999, 3333, 3001, 0, 9000], 3001, 4, 100),
        (8, 8, 4096, 64, [4096, 4095, 1025, 1024, 2047, 2100, 1, 4096], 1024, 0, 0),
        (4, 8, 4500, 128, [4500, 4097, 2500, 4400], 2500, 16, 1000),
        (33, 1, 2200, 128, [2200 - i for i in range(33)], 2100, 0, 2100),
        (12, 12, 1300, 32, [1300] * 11 + [650], 777, 1, 3),
        # selection of 16385 to 32768 rows, and one row past it
        (2, 2, 16385, 64, [16385, 16384], 5000, 4, 64),
        (3, 1, 20001, 32, [20001, 12000, 20000], 11999, 0, 0),
        (1, 3, 32768, 64, [32768], 32767, 7, 0),
        (2, 1, 32769, 32, [32769, 32768], 4096, 4, 1024),
        (2, 1, 16384, 32, [16384, 16001], 16000, 0, 5),
    ],
)
def test_evict_forms(gpu, B, Hk, cap, D, lens, keep, sinks, recent, dtype, layout):
    from SSA import ssa_cache_evict

    _say(f"evict form B={B} Hk={Hk} cap={cap} D={D} keep={keep} {dtype} {layout}")
    g = torch.Generator(device=gpu).manual_seed(keep)
    if layout == "bhsd":
        k, v = (_randn((B, Hk, cap, D), g, dtype, gpu) for _ in range(2))
    else:
        k, v = (_randn((B, cap, Hk, D), g, dtype, gpu).transpose(1, 2) for _ in range(2))
    w = _odd_weights(B, Hk, cap, cap, gpu)
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    new, left, kept = ssa_cache_evict(k, v, torch.tensor(lens, dtype=torch.int32, device=gpu), w, keep, sinks, recent)
    torch.cuda.synchronize()
    wn, wl, wk = _evicted(lens, w0, keep, sinks, recent)
    assert torch.equal(new, wn.int()) and torch.equal(kept, wk)
    assert torch.equal(left.view(torch.int32), wl.view(torch.int32))
    assert torch.equal(w.view(torch.int32), w0.view(torch.int32))
    rows = torch.arange(cap, device=gpu).expand(B, Hk, cap).clone()
    rows[..., :keep] = torch.where(wk >= 0, wk.long(), rows[..., :keep])
    for got, was in ((k, k0), (v, v0)):
        assert torch.equal(got, was.gather(2, rows[..., None].expand(-1, -1, -1, D)))
