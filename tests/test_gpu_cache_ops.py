"""The cache operators (SSA/ssa_cache_ops.py) against their definitions in 64 bits
(cache_ops_ref.py, which derives the bounds): trees, ragged and empty caches,
masks that leave nothing, values that must not be seen, strides, long offsets,
streams and graphs."""

from __future__ import annotations

import math
import sys

import pytest
import torch

import cache_ops_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _say(label):
    print(f"[gpu case] {label}", file=sys.stderr, flush=True)


def _randn(shape, gen, dtype, dev):
    return (torch.randn(shape, generator=gen)).to(dtype).to(dev)


def _caches(dev, B, Hk, cap, D, dtype, seed, layout="bhsd"):
    g = torch.Generator().manual_seed(seed)
    if layout == "bhsd":
        return _randn((B, Hk, cap, D), g, dtype, dev), _randn((B, Hk, cap, D), g, dtype, dev), g
    k, v = (_randn((B, cap, Hk, D), g, dtype, dev).transpose(1, 2) for _ in range(2))
    return k, v, g


def _scalars(dev, n=1.5, b=0.8):
    return torch.tensor(n, device=dev), torch.tensor(b, device=dev)


def _random_tree(T, seed, B=None):
    from SSA import tree_mask_from_parents

    g = torch.Generator().manual_seed(seed)
    one = lambda: [-1 if i == 0 else max(-1, i - int(torch.randint(1, 6, (1,), generator=g))) for i in range(T)]  # noqa: E731
    return tree_mask_from_parents([one() for _ in range(B)] if B else one())


def _check_tree(dev, q, k, v, lens, mask, n=1.5, b=0.8, splits=0):
    from SSA import ssa_tree_attention

    scale = 1.0 / math.sqrt(q.shape[-1])
    out, m = ssa_tree_attention(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), mask.to(dev), scale,
                                *_scalars(dev, n, b), num_splits=splits, return_m=True)
    torch.cuda.synchronize()
    want, wm, tol, mtol = ref.tree(q, k, v, lens, mask.to(dev), scale, n, b)
    off = (out.double() - want).abs()
    assert out.shape == q.shape and out.dtype == q.dtype
    assert bool((off <= tol).all()), f"out: {float((off - tol).max())} over its bound, error {float(off.max())}"
    empty = wm == -math.inf
    assert torch.equal(m == -math.inf, empty)
    moff = torch.where(empty, torch.zeros_like(wm), (m.double() - wm).abs())
    assert bool((moff <= mtol).all()), f"m: {float((moff - mtol).max())} over its bound"
    return out, m


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize(
    "B,Hq,Hk,cap,T,lens,splits",
    [
        (1, 4, 4, 64, 1, [64], 0),
        (2, 8, 2, 300, 7, [300, 45], 0),
        (3, 4, 4, 257, 32, [257, 32, 200], 3),       # 32 rows; a cache that is the tree alone
        (2, 6, 2, 500, 11, [500, 129], 0),           # 33 rows: two groups, the second with one row
        (2, 16, 4, 1000, 16, [1000, 640], 1),        # 64 rows, one split
        (1, 24, 8, 1000, 61, [999], 0),              # 183 rows
        (2, 8, 2, 700, 31, [700, 333], 0),           # 124 rows
        (1, 16, 1, 2100, 65, [2100], 0),             # 1040 rows: five blocks, T past 64
        (2, 2, 2, 900, 200, [900, 250], 2),          # a mask of several words
        (4, 8, 8, 96, 5, [0, 3, 5, 1000], 0),        # empty, shorter than the tree, the tree alone, past the capacity
    ],
)
def test_tree_matches_definition(gpu, D, dtype, B, Hq, Hk, cap, T, lens, splits):
    _say(f"tree D={D} {dtype} B={B} Hq={Hq} Hk={Hk} cap={cap} T={T} lens={lens} splits={splits}")
    k, v, g = _caches(gpu, B, Hk, cap, D, dtype, seed=D + T)
    q = _randn((B, Hq, T, D), g, dtype, gpu)
    _check_tree(gpu, q, k, v, lens, _random_tree(T, 5 * T, B if T % 2 else None), splits=splits)


def test_tree_largest(gpu):
    """1024 nodes, three heads a group, random masks."""
    _say("tree T=1024")
    k, v, g = _caches(gpu, 1, 1, 1500, 64, BF16, seed=2)
    q = _randn((1, 3, 1024, 64), g, BF16, gpu)
    mask = torch.rand(1024, 1024, generator=g) < 0.1
    _check_tree(gpu, q, k, v, [1400], mask)


@pytest.mark.parametrize("rows", [20, 60, 120, 300])
def test_tree_masks_that_leave_nothing(gpu, rows):
    """Nodes that see nothing in caches that hold the tree alone; a mask of zeros."""
    _say(f"tree empty rows={rows}")
    k, v, g = _caches(gpu, 2, 1, 400, 64, BF16, seed=rows)
    q = _randn((2, 1, rows, 64), g, BF16, gpu)
    mask = torch.rand(rows, rows, generator=g) < 0.3
    mask[::3] = False
    _check_tree(gpu, q, k, v, [rows, rows + 1], mask)
    out, m = _check_tree(gpu, q, k, v, [rows, rows // 2], torch.zeros(rows, rows, dtype=torch.bool))
    assert bool((out == 0).all()) and bool((m == -math.inf).all())


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("G,T", [(1, 20), (2, 31), (4, 30), (4, 64)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_tree_keeps_unseen_values_out(gpu, D, G, T, dtype):
    """NaN and infinities in branches that a node does not see and in rows behind
    the sequence reach no result; a value that is seen does."""
    _say(f"tree unseen D={D} G={G} T={T} {dtype}")
    B, cap, lens = 2, 300, [250, 100]
    k, v, g = _caches(gpu, B, 1, cap, D, dtype, seed=T)
    q = _randn((B, G, T, D), g, dtype, gpu)
    mask = _random_tree(T, T)
    bad = [T - 1, T - 2, T // 2]
    mask[:, bad] = False
    clean, cm = _check_tree(gpu, q, k, v, lens, mask)
    for i, L in enumerate(lens):
        for j, value in zip(bad, (math.nan, math.inf, -math.inf)):
            k[i, :, L - T + j] = value
            v[i, :, L - T + j] = value
        k[i, :, L:] = math.nan
        v[i, :, L:] = math.inf
    out, m = _check_tree(gpu, q, k, v, lens, mask)
    assert torch.equal(out, clean) and torch.equal(m, cm)
    # column 1 of node T - 2's value is +inf, column 3 of it -inf and column 5 NaN: those who see it get them
    k[:, :, :] = torch.nan_to_num(k.float(), 0.0, 0.0, 0.0).to(dtype)
    v[:, :, :] = torch.nan_to_num(v.float(), 0.0, 0.0, 0.0).to(dtype)
    mask[T // 3, T - 2] = True
    for i, L in enumerate(lens):
        v[i, :, L - T + T - 2, 1], v[i, :, L - T + T - 2, 3], v[i, :, L - T + T - 2, 5] = math.inf, -math.inf, math.nan
    out, _ = _check_seen(gpu, q, k, v, lens, mask)
    rows = torch.zeros(T, dtype=torch.bool)
    rows[T // 3] = True
    assert bool((out[:, :, rows, 1] == math.inf).all()) and bool((out[:, :, rows, 3] == -math.inf).all())
    assert bool(out[:, :, rows, 5].isnan().all()) and bool(out[:, :, ~rows].isfinite().all())
    keep = [c for c in range(D) if c not in (1, 3, 5)]
    assert bool(out[:, :, rows][..., keep].isfinite().all())


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("G,splits", [(1, 0), (1, 2), (2, 0), (2, 2), (4, 0), (4, 2)])
def test_tree_workgroups_of_more_rows(gpu, D, dtype, G, splits):
    """61, 122 and 244 rows on workgroups of 64, 128 and 256: 256 (sequence, kv-head)
    pairs, so that smaller ones would take more rounds of the GPU.  Empty rows,
    empty sequences, and NaN and infinities where nothing looks."""
    B, Hk, cap, T = 16, 16, 300, 61
    _say(f"tree D={D} {dtype} G={G} splits={splits} wide workgroups")
    lens = [300, 0, 1, 61, 60, 62, 299, 256, 257, 288, 317, 100, 150, 200, 250, 128]
    k, v, g = _caches(gpu, B, Hk, cap, D, dtype, seed=G + D)
    q = _randn((B, G * Hk, T, D), g, dtype, gpu)
    mask = _random_tree(T, G, B)
    mask[3, ::4] = False
    unseen = [T - 1, T // 2]
    mask[:, :, unseen] = False
    clean, cm = _check_tree(gpu, q, k, v, lens, mask, splits=splits)
    for i, L in enumerate(lens):
        for j, value in zip(unseen, (math.nan, math.inf)):
            if 0 <= min(L, cap) - T + j:
                k[i, :, min(L, cap) - T + j] = value
                v[i, :, min(L, cap) - T + j] = -value
        k[i, :, L:] = math.inf
        v[i, :, L:] = math.nan
    out, m = _check_tree(gpu, q, k, v, lens, mask, splits=splits)
    assert torch.equal(out, clean) and torch.equal(m, cm)


def _check_seen(dev, q, k, v, lens, mask):
    from SSA import ssa_tree_attention

    r = ssa_tree_attention(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), mask.to(dev),
                           1.0 / math.sqrt(q.shape[-1]), *_scalars(dev), return_m=True)
    torch.cuda.synchronize()
    return r


@pytest.mark.parametrize("n,b", [(0.0, 0.8), (-3.5, 0.8), (5.0, 0.8), (1.5, 0.0), (-302.0, 0.8), (1e-30, 0.8)])
@pytest.mark.parametrize("T", [9, 40, 100])
def test_tree_and_weights_scalars(gpu, n, b, T):
    """n of both signs, 0 and tiny, b = 0; queries whose exponents lie far below 0."""
    _say(f"tree and weights n={n} b={b} T={T}")
    k, v, g = _caches(gpu, 1, 2, 400, 64, BF16, seed=7)
    q = _randn((1, 4, T, 64), g, BF16, gpu)
    _check_tree(gpu, q, k, v, [400], _random_tree(T, 3), n=n, b=b)
    _check_weights(gpu, q, k, [400], n=n, b=b)


@pytest.mark.parametrize("T", [5, 30, 70])
def test_tree_strides(gpu, T):
    """[T, B, H, D] queries and [B, cap, H, D] caches as views; masks of other types; q as [B, H, D]."""
    from SSA import ssa_tree_attention

    _say(f"tree strides T={T}")
    k, v, g = _caches(gpu, 2, 2, 333, 64, BF16, seed=T, layout="bshd")
    q = _randn((T, 2, 4, 64), g, BF16, gpu).permute(1, 2, 0, 3)
    mask = _random_tree(T, T)
    out, m = _check_tree(gpu, q, k, v, [333, 100], mask)
    lens = torch.tensor([333, 100], device=gpu)
    args = (k, v, lens, mask.to(gpu).float(), 0.125, 1.5, 0.8)
    got = ssa_tree_attention(q.transpose(2, 3).contiguous().transpose(2, 3), *args)
    assert torch.equal(got, out)
    got = ssa_tree_attention(q, k, v, [333, 100], mask.tolist(), 0.125, 1.5, 0.8)
    assert torch.equal(got, out)
    one, m1 = ssa_tree_attention(q[:, :, 0], k, v, lens, torch.ones(1, 1), 0.125, 1.5, 0.8, return_m=True)
    assert one.shape == (2, 4, 64) and m1.shape == (2, 4)


def test_tree_of_one_is_the_decode_step(gpu):
    from SSA import ssa_decode_attention, ssa_tree_attention

    _say("tree of one node")
    k, v, g = _caches(gpu, 3, 4, 700, 128, BF16, seed=4)
    q = _randn((3, 16, 128), g, BF16, gpu)
    lens = torch.tensor([700, 1, 333], dtype=torch.int32, device=gpu)
    out, m = ssa_tree_attention(q, k, v, lens, torch.ones(1, 1, dtype=torch.bool, device=gpu), 0.088, 1.5, 0.8,
                                return_m=True)
    want, wm = ssa_decode_attention(q, k, v, lens, 0.088, 1.5, 0.8, return_m=True)
    # each is within a half step of rounding, twice (out and p), of the same value
    assert bool(((out.float() - want.float()).abs() <= 2.0 ** -6 * want.float().abs().clamp_min(0.25)).all())
    assert bool(((m - wm).abs() <= 2.0 ** -15).all())


def test_tree_reproducible_and_per_sequence(gpu):
    """Bitwise: run to run, and a sequence's result whatever the others hold."""
    from SSA import ssa_tree_attention

    _say("tree reproducible")
    k, v, g = _caches(gpu, 4, 2, 2048, 64, BF16, seed=9)
    q = _randn((4, 8, 24, 64), g, BF16, gpu)
    mask = _random_tree(24, 1).to(gpu)
    lens = torch.tensor([2048, 24, 900, 1500], dtype=torch.int32, device=gpu)
    a = ssa_tree_attention(q, k, v, lens, mask, 0.125, 1.5, 0.8, return_m=True)
    b = ssa_tree_attention(q, k, v, lens, mask, 0.125, 1.5, 0.8, return_m=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    lens[1], lens[3] = 0, 31
    c = ssa_tree_attention(q, k, v, lens, mask, 0.125, 1.5, 0.8, return_m=True)
    assert torch.equal(a[0][[0, 2]], c[0][[0, 2]]) and torch.equal(a[1][[0, 2]], c[1][[0, 2]])


# ------------------------------------------------------------------ key weights
def _normalisers(q, k, lens, scale, n, b):
    B, Hq, T, _ = q.shape
    m = torch.full((B, Hq, T), -math.inf, device=q.device)
    for i in range(B):
        L = min(max(int(lens[i]), 0), k.shape[2])
        seen = (torch.arange(L, device=q.device)[None, :] <= torch.arange(L - T, L, device=q.device)[:, None])
        for h in range(Hq):
            t = ref.transform(scale * (q[i, h].double() @ k[i, h // (Hq // k.shape[1]), :L].double().t()), n, b)
            t = t.masked_fill(~seen, -math.inf)
            if L:
                m[i, h] = ((t * ref.LN2).logsumexp(1) / ref.LN2).float()
    return m


def _check_weights(dev, q, k, lens, n=1.5, b=0.8, m=None, weights=None):
    from SSA import ssa_key_weights

    scale = 1.0 / math.sqrt(q.shape[-1])
    m = _normalisers(q, k, lens, scale, n, b) if m is None else m
    if weights is None:
        weights = torch.rand(k.shape[:3], device=dev)
    before = weights.clone()
    got = ssa_key_weights(q, k, m, torch.tensor(lens, dtype=torch.int32, device=dev), weights, scale,
                          *_scalars(dev, n, b))
    torch.cuda.synchronize()
    assert got is weights
    want, tol = ref.key_weights(q, k, m, lens, before, scale, n, b)
    for i, L in enumerate(lens):
        L = min(max(L, 0), k.shape[2])
        assert torch.equal(weights[i, :, L:], before[i, :, L:])  # rows behind the sequence stay
        off = (weights[i, :, :L].double() - want[i, :, :L]).abs()
        assert bool((off <= tol[i, :, :L]).all()), f"{float((off - tol[i, :, :L]).max())} over the bound"
    return weights


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize(
    "B,Hq,Hk,cap,T,lens",
    [
        (1, 4, 4, 64, 1, [64]),
        (3, 8, 2, 300, 1, [300, 1, 130]),
        (2, 32, 1, 200, 1, [200, 77]),            # 32 rows
        (2, 33, 1, 200, 1, [200, 77]),            # 33
        (2, 6, 2, 700, 13, [700, 13]),            # 39 rows, three heads a group; a cache of the queries alone
        (2, 8, 8, 513, 32, [513, 100]),
        (1, 16, 4, 1000, 100, [1000]),
        (2, 4, 4, 300, 300, [300, 300]),          # a whole prompt
        (1, 24, 8, 777, 777, [777]),
        (4, 4, 2, 128, 20, [0, 7, 20, 500]),      # empty, shorter than the queries, past the capacity
    ],
)
def test_weights_match_definition(gpu, D, dtype, B, Hq, Hk, cap, T, lens):
    _say(f"weights D={D} {dtype} B={B} Hq={Hq} Hk={Hk} cap={cap} T={T} lens={lens}")
    k, _, g = _caches(gpu, B, Hk, cap, D, dtype, seed=D + T)
    _check_weights(gpu, _randn((B, Hq, T, D), g, dtype, gpu), k, lens)


@pytest.mark.parametrize("T", [3, 90])
def test_weights_rows_that_add_nothing(gpu, T):
    """Queries whose m is -inf, NaN queries among them, and NaN keys behind the
    sequence or the query; negative and zero n."""
    _say(f"weights -inf rows T={T}")
    k, _, g = _caches(gpu, 2, 2, 300, 64, BF16, seed=T)
    q = _randn((2, 4, T, 64), g, BF16, gpu)
    lens = [299, 200]
    for n in (1.5, -2.0, 0.0):
        m = _normalisers(q, k, lens, 0.125, n, 0.8)
        m[:, 1, T // 2] = -math.inf
        _check_weights(gpu, q, k, lens, n=n, m=m)
    m = _normalisers(q, k, lens, 0.125, 1.5, 0.8)
    m[:, 1, T // 2] = -math.inf
    want = _check_weights(gpu, q, k, lens, m=m, weights=torch.zeros(2, 2, 300, device=gpu))
    q[:, 1, T // 2] = math.nan
    k[0, :, 299:] = math.nan
    k[1, :, 200:] = math.inf
    from SSA import ssa_key_weights

    w = torch.zeros(2, 2, 300, device=gpu)
    ssa_key_weights(q, k, m, torch.tensor(lens, dtype=torch.int32, device=gpu), w, 0.125, 1.5, 0.8)
    assert torch.equal(w, want)
    # the last cached key is NaN: it alone is NaN, for the queries before it do not see it
    k[0, :, 298] = math.nan
    w = torch.zeros(2, 2, 300, device=gpu)
    ssa_key_weights(q, k, m, torch.tensor(lens, dtype=torch.int32, device=gpu), w, 0.125, 1.5, 0.8)
    assert torch.equal(w[0, :, :298], want[0, :, :298]) and bool(w[0, :, 298].isnan().all())


def test_weights_strides_and_sums(gpu):
    """Strided weights, queries and caches; the probabilities of a query add up to 1."""
    from SSA import ssa_flash_attn_forward, ssa_key_weights

    _say("weights strides")
    k, _, g = _caches(gpu, 2, 2, 260, 64, BF16, seed=3, layout="bshd")
    q = _randn((40, 2, 4, 64), g, BF16, gpu).permute(1, 2, 0, 3)
    room = torch.zeros(2, 2, 300, device=gpu)
    _check_weights(gpu, q, k, [260, 100], weights=room[..., :260])
    assert bool((room[..., 260:] == 0).all())
    L = 200
    qf = _randn((2, 4, L, 64), g, BF16, gpu)
    kf, vf = k[:, :, :L], k[:, :, :L]
    _, m = ssa_flash_attn_forward(qf, kf, vf, 0.125, torch.tensor(1.5, device=gpu), torch.tensor(0.8, device=gpu))
    w = torch.zeros(2, 2, 260, device=gpu)
    ssa_key_weights(qf, k, m, [L, L], w, 0.125, 1.5, 0.8)
    # 2 heads a group, 200 queries each, of probability 1; m comes from the forward's own fp32 sums
    assert torch.allclose(w.sum(-1), torch.full((2, 2), 2.0 * L, device=gpu), rtol=2.0 ** -12)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,Hq,Hk,cap,T,lens", [
    (2, 4, 4, 1000, 65, [1000, 64]),        # 65 rows on few workgroups: two waves of rows
    (2, 8, 2, 257, 100, [257, 30]),         # 400 rows
    (16, 16, 16, 1024, 65, [1024, 1000, 65, 64, 1, 0, 129, 128] * 2),  # 2048 workgroups: one wave
    (16, 32, 16, 1024, 300, [1024, 1000, 300, 299, 1, 0, 513, 512] * 2),  # ... of 600 rows: two
])
def test_weights_of_either_form(gpu, D, B, Hq, Hk, cap, T, lens):
    _say(f"weights D={D} B={B} Hq={Hq} Hk={Hk} cap={cap} T={T}")
    k, _, g = _caches(gpu, B, Hk, cap, D, BF16, seed=D + T)
    _check_weights(gpu, _randn((B, Hq, T, D), g, BF16, gpu), k, lens)


def test_weights_of_chunks_that_do_not_divide(gpu):
    """Rows split into chunks that whole stages make longer than an even share;
    the workspace comes from memory that held NaN."""
    B, Hq, Hk, cap, T, D = 1, 32, 1, 1280, 1200, 32
    _say("weights of 38400 rows in chunks that do not divide them")
    k, _, g = _caches(gpu, B, Hk, cap, D, BF16, seed=11)
    q = _randn((B, Hq, T, D), g, BF16, gpu)
    for chunks in range(30, 80):
        torch.full((chunks * cap,), math.nan, device=gpu)  # freed at once, for the next of its size
    _check_weights(gpu, q, k, [1250])


# ------------------------------------------------------------------------ evict
def _check_evict(dev, lens, weights, keep, sinks, recent, D=64, dtype=BF16, layout="bhsd"):
    from SSA import ssa_cache_evict

    B, Hk, cap = weights.shape
    k, v, _ = _caches(dev, B, Hk, cap, D, dtype, seed=keep, layout=layout)
    k0, v0, w0 = k.clone(), v.clone(), weights.clone()
    lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
    new, left, kept = ssa_cache_evict(k, v, lens_t, weights, keep, sinks=sinks, recent=recent)
    torch.cuda.synchronize()
    wn, wl, wk = ref.evict(lens, weights, keep, sinks, recent)
    assert new.tolist() == wn and lens_t.tolist() == list(lens)
    assert torch.equal(kept.cpu(), wk)
    assert torch.equal(left.cpu().view(torch.int32), wl.view(torch.int32))
    assert torch.equal(weights.view(torch.int32), w0.view(torch.int32))
    for i in range(B):
        for h in range(Hk):
            rows = wk[i, h, :wn[i]].long().to(dev)
            assert torch.equal(k[i, h, :wn[i]], k0[i, h, rows]) and torch.equal(v[i, h, :wn[i]], v0[i, h, rows])
            assert torch.equal(k[i, h, wn[i]:], k0[i, h, wn[i]:]) and torch.equal(v[i, h, wn[i]:], v0[i, h, wn[i]:])


@pytest.mark.parametrize(
    "cap,lens,keep,sinks,recent",
    [
        (64, [64, 10], 32, 4, 8),
        (500, [500, 499, 251, 250, 0, 900], 250, 4, 100),
        (1000, [1000], 1, 0, 0),
        (1000, [1000, 1000], 1, 1, 0),
        (1000, [1000, 800], 999, 0, 999),
        (1000, [1000], 1000, 10, 20),
        (5000, [5000, 4097], 1234, 0, 0),        # more than one stretch of the selection
        (9000, [9000], 8999, 16, 1000),
        (2050, [2050, 2050], 2049, 0, 7),
        (300, [300, 300], 100, 40, 60),          # nothing to choose
    ],
)
def test_evict_matches_definition(gpu, cap, lens, keep, sinks, recent):
    _say(f"evict cap={cap} lens={lens} keep={keep} sinks={sinks} recent={recent}")
    g = torch.Generator().manual_seed(cap)
    w = torch.randn(len(lens), 2, cap, generator=g).mul(1.5).exp().to(gpu)
    _check_evict(gpu, lens, w, keep, sinks, recent)


def test_evict_equal_and_odd_weights(gpu):
    """Equal weights (the lower rows stay), zeros of both signs, infinities, NaN of
    both signs, denormals and negative weights."""
    _say("evict odd weights")
    g = torch.Generator().manual_seed(1)
    cap = 700
    w = torch.zeros(6, 2, cap)
    w[0] = 1.0
    w[1] = torch.randint(0, 3, (2, cap), generator=g).float()
    w[2] = torch.tensor([0.0, -0.0, 1e-40, -1e-40])[torch.randint(0, 4, (2, cap), generator=g)]
    w[3] = torch.tensor([math.inf, -math.inf, math.nan, 1.0])[torch.randint(0, 4, (2, cap), generator=g)]
    w[4] = torch.randn(2, cap, generator=g)
    w[5] = math.nan
    w[5, 1, ::2] = -math.nan
    for keep in (100, 351, 650):
        _check_evict(gpu, [cap] * 6, w.to(gpu), keep, 3, 50)


@pytest.mark.parametrize("D,dtype,layout", [(32, BF16, "bshd"), (128, FP16, "bhsd"), (128, BF16, "bshd")])
def test_evict_layouts(gpu, D, dtype, layout):
    _say(f"evict D={D} {dtype} {layout}")
    g = torch.Generator().manual_seed(D)
    room = torch.rand(2, 3, 1300, generator=g).to(gpu)
    _check_evict(gpu, [1290, 1000], room[..., :1290], 600, 4, 16, D, dtype, layout)


def test_evict_long_cache(gpu):
    _say("evict 70000 rows")
    g = torch.Generator().manual_seed(6)
    w = torch.rand(1, 1, 70000, generator=g).pow(8).to(gpu)
    _check_evict(gpu, [70000], w, 30000, 4, 64, 32)


# ----------------------------------------------------------------------- accept
def _check_accept(dev, lens, path, accepted, nodes, cap, Hk=2, D=64, dtype=BF16, layout="bhsd"):
    from SSA import ssa_cache_accept

    B = len(lens)
    k, v, _ = _caches(dev, B, Hk, cap, D, dtype, seed=nodes, layout=layout)
    wk, wv = k.clone(), v.clone()
    lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
    new = ssa_cache_accept(k, v, lens_t, torch.tensor(path, dtype=torch.int32, device=dev),
                           torch.tensor(accepted, dtype=torch.int32, device=dev), nodes)
    torch.cuda.synchronize()
    want = []
    for i, L in enumerate(lens):
        L = min(max(L, 0), cap)
        first = L - nodes
        if first < 0:
            want.append(L)
            continue
        n = min(max(accepted[i], 0), len(path[i]))
        want.append(first + n)
        at = [first + min(max(x, 0), nodes - 1) for x in path[i][:n]]
        for c in (wk, wv):
            c[i, :, first:first + n] = c[i, :, at].clone()
    assert new.tolist() == want and lens_t.tolist() == list(lens)
    assert torch.equal(k, wk) and torch.equal(v, wv)


@pytest.mark.parametrize("D,dtype,layout", [(32, BF16, "bhsd"), (64, FP16, "bshd"), (128, BF16, "bhsd")])
def test_accept_matches_definition(gpu, D, dtype, layout):
    _say(f"accept D={D} {dtype} {layout}")
    g = torch.Generator().manual_seed(D)
    for nodes, depth in ((1, 1), (8, 3), (64, 17), (200, 200), (1024, 1024), (1024, 5)):
        path = [sorted(torch.randperm(nodes, generator=g)[:depth].tolist()) for _ in range(5)]
        lens = [nodes, nodes + 100, nodes + 1, nodes - 1, 5000]
        _check_accept(gpu, lens, path, [depth, depth // 2, 0, 1, depth], nodes, 1200, D=D, dtype=dtype, layout=layout)


def test_accept_any_order_and_clamps(gpu):
    """A path that is not ascending, one node twice, nodes and counts out of range."""
    _say("accept any order")
    g = torch.Generator().manual_seed(8)
    path = [torch.randperm(300, generator=g).tolist() for _ in range(2)]
    path += [[299] * 300, [-5, 400, 2 ** 31 - 1, -2 ** 31] * 75]
    _check_accept(gpu, [300, 500, 500, 400], path, [300, 299, 1000, 300], 300, 600)
    _check_accept(gpu, [300, 500], path[:2], [-3, 2 ** 31 - 1], 300, 600)


# -------------------------------------------------------- offsets, streams, graphs
def test_offsets_past_32_bits(gpu):
    """Caches whose elements lie past 2^32 bytes from their base."""
    from SSA import ssa_cache_accept, ssa_cache_evict, ssa_key_weights, ssa_tree_attention

    _say("offsets past 2^32 bytes")
    cap, D, step = 700, 64, 1 << 22  # 2.9e9 elements
    room = torch.zeros(cap * step + D, dtype=BF16, device=gpu)
    far = room.as_strided((1, 1, cap, D), (0, 0, step, 1))
    k, v, g = _caches(gpu, 1, 1, cap, D, BF16, seed=12)
    far.copy_(k)
    q = _randn((1, 2, 40, D), g, BF16, gpu)
    mask = _random_tree(40, 2).to(gpu)
    lens = torch.tensor([cap], dtype=torch.int32, device=gpu)
    for T in (8, 24, 40):
        a = ssa_tree_attention(q[:, :, :T], k, k.clone(), lens, mask[:T, :T], 0.125, 1.5, 0.8, return_m=True)
        b = ssa_tree_attention(q[:, :, :T], far, far, lens, mask[:T, :T], 0.125, 1.5, 0.8, return_m=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    w = torch.zeros(2, 1, 1, cap, device=gpu)
    ssa_key_weights(q, k, a[1], lens, w[0], 0.125, 1.5, 0.8)
    ssa_key_weights(q, far, a[1], lens, w[1], 0.125, 1.5, 0.8)
    assert torch.equal(w[0], w[1])
    path, count = torch.tensor([[3, 9, 30]], device=gpu), torch.tensor([3], device=gpu)
    v2 = v.clone()
    ssa_cache_accept(k, v, lens, path, count, 40)
    ssa_cache_accept(far, v2, lens, path, count, 40)
    assert torch.equal(k, far) and torch.equal(v, v2)
    ssa_cache_evict(k, v, lens, w[0], 300, sinks=4, recent=16)
    ssa_cache_evict(far, v2, lens, w[0], 300, sinks=4, recent=16)
    assert torch.equal(k, far) and torch.equal(v, v2)


def _round(q, k, v, lens, mask, path, count, w, n, b):
    """Draft, accept, weigh and cut: one turn of a generation loop; everything it returns."""
    from SSA import ssa_cache_accept, ssa_cache_evict, ssa_key_weights, ssa_tree_attention

    T = q.shape[2]
    out, m = ssa_tree_attention(q, k, v, lens, mask, 0.125, n, b, return_m=True)
    new = ssa_cache_accept(k, v, lens, path, count, T)
    A = path.shape[1]
    at = path.long()[:, None, :].expand(-1, q.shape[1], -1)
    ssa_key_weights(q.gather(2, at[..., None].expand(-1, -1, -1, q.shape[3])), k, m.gather(2, at), new, w, 0.125, n, b)
    lens2, w2, kept = ssa_cache_evict(k, v, new, w, 200, sinks=2, recent=A)
    return out, m, new, lens2, w2, kept


def _round_inputs(dev, seed, rows=24):
    k, v, g = _caches(dev, 2, 2, 512, 64, BF16, seed=seed)
    q = _randn((2, 8, rows, 64), g, BF16, dev)
    mask = _random_tree(rows, seed).to(dev)
    path = torch.tensor([[0, 2, 5, 9], [1, 3, 4, 11]], dtype=torch.int32, device=dev)
    count = torch.tensor([4, 4], dtype=torch.int32, device=dev)
    lens = torch.tensor([500, 300], dtype=torch.int32, device=dev)
    return q, k, v, lens, mask, path, count, torch.rand(2, 2, 512, generator=g).to(dev), *_scalars(dev)


@pytest.mark.parametrize("rows", [4 + 8, 32])
def test_whole_turn_against_definitions(gpu, rows):
    """A turn of draft, acceptance, weights and eviction, step by step."""
    _say(f"whole turn rows={rows}")
    q, k, v, lens, mask, path, count, w, n, b = _round_inputs(gpu, 3, rows)
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    out, m, new, lens2, w2, kept = _round(q, k, v, lens, mask, path, count, w, n, b)
    torch.cuda.synchronize()
    want, wm, tol, mtol = ref.tree(q, k0, v0, lens.tolist(), mask, 0.125, 1.5, 0.8)
    assert bool(((out.double() - want).abs() <= tol).all()) and bool(((m.double() - wm).abs() <= mtol).all())
    for i in range(2):
        first = int(lens[i]) - rows
        at = [first + x for x in path[i].tolist()]
        k0[i, :, first:first + 4], v0[i, :, first:first + 4] = k0[i, :, at].clone(), v0[i, :, at].clone()
    after = [int(x) - rows + 4 for x in lens]
    assert new.tolist() == after
    index = path.long()[:, None, :].expand(-1, 8, -1)
    qa, ma = q.gather(2, index[..., None].expand(-1, -1, -1, 64)), m.gather(2, index)
    ww, wtol = ref.key_weights(qa, k0, ma, after, w0, 0.125, 1.5, 0.8)
    assert bool(((w.double() - ww).abs() <= wtol).all())
    wn, wl, wk = ref.evict(after, w, 200, 2, 4)
    assert lens2.tolist() == wn and torch.equal(kept.cpu(), wk) and torch.equal(w2.cpu(), wl)
    for i in range(2):
        for h in range(2):
            r = wk[i, h].long().to(gpu)
            assert torch.equal(k[i, h, :200], k0[i, h, r]) and torch.equal(v[i, h, :200], v0[i, h, r])


def test_side_stream_and_two_at_once(gpu):
    """Two turns on two streams at once give what they give alone."""
    _say("two streams")
    alone = [_round(*_round_inputs(gpu, s)) for s in (1, 2)]
    states = [_round_inputs(gpu, s) for s in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, st in zip(streams, states):
        with torch.cuda.stream(s):
            got.append(_round(*st))
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_turns(gpu):
    """Two captured turns replayed in turn, with other work between, give the eager results each time."""
    _say("captured turns")
    states = [_round_inputs(gpu, s) for s in (4, 5)]
    saved = [[t.clone() for t in st] for st in states]
    eager = [[x.clone() for x in _round(*[t.clone() for t in st])] for st in states]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for st in states:
            _round(*[t.clone() for t in st])
    torch.cuda.current_stream().wait_stream(side)
    for st in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_round(*st))
        graphs.append(graph)
    for turn in range(3):
        for i in (0, 1):
            for t, s in zip(states[i], saved[i]):
                t.copy_(s)
            _round(*[t.clone() for t in saved[1 - i]])  # eager work in between
            graphs[i].replay()
            torch.cuda.synchronize()
            for x, y in zip(outs[i], eager[i]):
                assert torch.equal(x, y), f"turn {turn} graph {i}"


def test_native_and_python_paths_agree(gpu, monkeypatch):
    """The extension module's path and the Python path give the same bits."""
    from SSA import _lib

    _say("native against Python path")
    native = _round(*_round_inputs(gpu, 6))
    monkeypatch.setattr(_lib, "native", lambda: _lib.PythonPath())
    python = _round(*_round_inputs(gpu, 6))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(native, python))
