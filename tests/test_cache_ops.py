"""The cache operators' checks of arguments, without a GPU: the C ABI's
(include/ssa_cache_ops.h), where every call is rejected before any launch, and
the Python layer's."""

from __future__ import annotations

import ctypes

import pytest
import torch

from SSA import _lib

FAKE = 1 << 20  # an aligned address that is never read
N, A, H, D, S = (_lib.SSA_ERR_NULL_POINTER, _lib.SSA_ERR_ALIGNMENT, _lib.SSA_ERR_HEAD_DIM, _lib.SSA_ERR_DTYPE,
                 _lib.SSA_ERR_SHAPE)


def _cache():
    return _lib.Tensor4(FAKE, 8 * 4096 * 64, 4096 * 64, 64)


def _other():
    return _lib.Tensor4(FAKE << 10, 8 * 4096 * 64, 4096 * 64, 64)


def _tree(**kw):
    q = _lib.Tensor4(FAKE, 32 * 16 * 64, 16 * 64, 64)
    a = _lib.TreeArgs(q, _cache(), _other(), q, None, FAKE, FAKE, 0, FAKE, FAKE, 4, 32, 8, 4096, 64,
                      _lib.SSA_DTYPE_BF16, 16, 0, 0.125, FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _weights(**kw):
    q = _lib.Tensor4(FAKE, 32 * 16 * 64, 16 * 64, 64)
    a = _lib.KeyWeightsArgs(q, _cache(), FAKE, FAKE, 8 * 4096, 4096, FAKE, FAKE, FAKE, 4, 32, 8, 4096, 64,
                            _lib.SSA_DTYPE_BF16, 16, 0.125, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _evict(**kw):
    a = _lib.CacheEvictArgs(_cache(), _other(), FAKE, 8 * 4096, 4096, FAKE, FAKE + 64, FAKE + 4096, FAKE, 4, 8, 4096,
                            64, _lib.SSA_DTYPE_BF16, 1024, 4, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _accept(**kw):
    a = _lib.CacheAcceptArgs(_cache(), _other(), FAKE, FAKE, FAKE, FAKE + 64, 4, 8, 4096, 64, _lib.SSA_DTYPE_FP16, 16,
                             5)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


CASES = [
    ("ssa_tree_attention", _tree, [
        ("batch", 0, S), ("heads_kv", 5, S), ("capacity", 0, S), ("capacity", (1 << 30) + 1, S), ("nodes", 0, S),
        ("nodes", 1025, S), ("num_splits", -1, S), ("batch", 1 << 28, S), ("head_dim", 48, H), ("head_dim", 256, H),
        ("dtype", _lib.SSA_DTYPE_FP32, D), ("dtype", 7, D), ("q", _lib.Tensor4(None, 0, 0, 64), N),
        ("q", _lib.Tensor4(FAKE + 2, 0, 0, 64), A), ("k_cache", _lib.Tensor4(FAKE, 0, 0, 60), A),
        ("v_cache", _lib.Tensor4(FAKE, 0, -64, 64), A), ("v_cache", _lib.Tensor4(FAKE, 0, 0, 1 << 24), A),
        ("out", _lib.Tensor4(FAKE + 8, 0, 0, 64), A), ("cache_seqlens", None, N), ("tree_mask", None, N),
        ("ssa_n", None, N), ("ssa_b", None, N), ("mask_stride_b", -1, A), ("workspace", None, N),
        ("workspace", FAKE + 8, A)]),
    ("ssa_key_weights", _weights, [
        ("batch", -1, S), ("heads_q", 31, S), ("queries", 0, S), ("queries", 4097, S), ("capacity", 0, S),
        ("head_dim", 16, H), ("dtype", _lib.SSA_DTYPE_FP32, D), ("q", _lib.Tensor4(FAKE + 4, 0, 0, 64), A),
        ("k_cache", _lib.Tensor4(None, 0, 0, 64), N), ("m", None, N), ("weights", None, N), ("weights", FAKE + 2, A),
        ("m", FAKE + 1, A), ("weights_stride_h", 4095, A), ("weights_stride_b", 0, A), ("weights_stride_h", -4096, A),
        ("cache_seqlens", None, N), ("ssa_n", None, N), ("ssa_b", None, N)]),
    ("ssa_cache_evict", _evict, [
        ("keep", 0, S), ("keep", 4097, S), ("sinks", -1, S), ("recent", -1, S), ("recent", 1021, S),
        ("sinks", 2 ** 31 - 1, S), ("capacity", 512, S), ("head_dim", 256, H), ("dtype", 5, D),
        ("k_cache", _lib.Tensor4(None, 0, 0, 64), N), ("k_cache", _lib.Tensor4(FAKE, 0, 4096 * 64, 64), A),
        ("k_cache", _lib.Tensor4(FAKE, 8 * 4096 * 64, 4096 * 64, 56), A), ("v_cache", _cache(), A),
        ("weights", None, N), ("seqlens_out", None, N), ("seqlens_out", FAKE, A), ("weights_out", FAKE, A),
        ("kept", None, N), ("kept", FAKE + 1, A), ("cache_seqlens", None, N), ("weights_stride_b", -4, A)]),
    ("ssa_cache_accept", _accept, [
        ("nodes", 0, S), ("nodes", 1025, S), ("depth", 0, S), ("depth", 17, S), ("heads_kv", 0, S),
        ("head_dim", 96, H), ("dtype", _lib.SSA_DTYPE_FP32, D), ("v_cache", _cache(), A),
        ("v_cache", _lib.Tensor4(FAKE << 10, 8 * 4096 * 64, 0, 64), A), ("path", None, N), ("accepted", None, N),
        ("seqlens_out", None, N), ("seqlens_out", FAKE, A), ("cache_seqlens", None, N)]),
]


@pytest.mark.parametrize("entry,make,field,value,status",
                         [(e, m, *row) for e, m, rows in CASES for row in rows])
def test_rejected_before_launch(entry, make, field, value, status):
    assert getattr(_lib.lib(), entry)(ctypes.byref(make(**{field: value})), None) == status


@pytest.mark.parametrize("entry", [c[0] for c in CASES])
def test_null_args(entry):
    assert getattr(_lib.lib(), entry)(None, None) == N


def test_weights_workspace():
    """Only many rows of few heads are split: a float per cached row and chunk."""
    f = _lib.lib().ssa_key_weights_workspace_bytes
    assert f(16, 32, 8, 4096, 1) == 0 and f(4, 16, 16, 8192, 32) == 0
    n = f(1, 32, 8, 4096, 4096)
    assert n > 0 and n % (8 * 4096 * 4) == 0
    assert f(1, 32, 8, 4096, 4097) == 0 and f(0, 32, 8, 4096, 1) == 0 and f(1, 32, 5, 4096, 1) == 0
    a = _weights(batch=1, queries=4096)
    assert _lib.lib().ssa_key_weights(ctypes.byref(a), None) == N
    a.workspace = FAKE + 4
    assert _lib.lib().ssa_key_weights(ctypes.byref(a), None) == A


@pytest.mark.parametrize("heads,T,cap", [(32, 1200, 1280), (32, 4000, 4096), (24, 3000, 3000), (7, 1000, 1000)])
def test_weights_chunks_all_hold_rows(heads, T, cap):
    """No chunk of the rows is empty: its part of the workspace would be added
    up without having been written."""
    chunks = _lib.lib().ssa_key_weights_workspace_bytes(1, heads, 1, cap, T) // (cap * 4)
    rows = heads * T
    # chunks of one length that is whole stages of 64 rows, 512 rows or more: some
    # length makes that many of them without an empty one
    assert chunks >= 2
    assert any((rows + per - 1) // per == chunks for per in range(512, rows + 64, 64))


def test_weights_of_groups_past_int32():
    """The first row that sees the last key of a tile is counted with 32 bits: up to
    128 queries past the last, times the heads of a group."""
    f = _lib.lib().ssa_key_weights
    q = _lib.Tensor4(FAKE, 0, 0, 64)
    for heads, queries, status in [(1 << 29, 1, S), (1 << 24, 1, S), (1 << 23, 128, S), (1 << 23, 64, N)]:
        a = _weights(batch=1, heads_q=heads, heads_kv=1, queries=queries, q=q, m=None)
        assert f(ctypes.byref(a), None) == status
        assert status == N or _lib.lib().ssa_key_weights_workspace_bytes(1, heads, 1, 4096, queries) == 0


def test_tree_splits_and_workspace():
    lib = _lib.lib()
    n, w = lib.ssa_tree_num_splits, lib.ssa_tree_workspace_bytes
    assert n(16, 16, 16, 4096, 64, 0) == 1 and w(16, 16, 16, 4096, 128, 64, 0) == 0  # 256 workgroups already
    assert n(1, 16, 16, 2048, 8, 0) == 8      # at least 256 keys a split
    assert n(1, 16, 16, 2048, 8, 3) == 3 and n(1, 16, 16, 2048, 8, 1000) == 8
    assert n(1, 16, 16, 200, 8, 0) == 1 and n(1, 16, 16, 200, 8, 5) == 1
    recs = 16 * 8 * 8
    assert w(1, 16, 16, 2048, 128, 8, 0) == (2 * recs + recs * 128) * 4
    for bad in ((0, 8, 8, 64, 4, 0), (1, 8, 3, 64, 4, 0), (1, 8, 8, 0, 4, 0), (1, 8, 8, 64, 0, 0), (1, 8, 8, 64, 4, -1)):
        assert n(*bad) == 0 and w(*bad[:4], 64, *bad[4:]) == 0
    assert w(1, 8, 8, 4096, 96, 4, 0) == 0


def test_default_splits_of_any_capacity():
    """At most one split per 256 rows, whatever the sizes; 0 beyond the limits."""
    lib = _lib.lib()
    for cap in [1, 255, 256, 257, 1000, 4096, 5000, 65536, 100001, 1 << 30]:
        for B, Hq, Hk, T in [(1, 8, 8, 1), (4, 32, 8, 33), (1, 16, 1, 64), (300, 4, 4, 5)]:
            s = lib.ssa_tree_num_splits(B, Hq, Hk, cap, T, 0)
            if s == 0:
                assert B * Hk * ((cap + 127) // 128) > 1 << 28
            else:
                assert 1 <= s <= (cap + 255) // 256


# ------------------------------------------------------------- the Python layer
def _cpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_python_refuses_host_tensors_and_wrong_shapes():
    from SSA import ssa_cache_accept, ssa_cache_evict, ssa_key_weights, ssa_tree_attention

    k, q = _cpu(2, 2, 64, 64), _cpu(2, 4, 5, 64)
    lens, mask = torch.tensor([64, 10]), torch.ones(5, 5)
    for bad in (k, _cpu(2, 64, 64), None, _cpu(2, 2, 64, 64, dtype=torch.float32)):
        with pytest.raises(ValueError):
            ssa_tree_attention(q, bad, bad, lens, mask, 0.1, 1.5, 0.8)
    with pytest.raises(ValueError):
        ssa_key_weights(q, k, torch.zeros(2, 4, 5), lens, torch.zeros(2, 2, 64), 0.1, 1.5, 0.8)
    with pytest.raises(ValueError):
        ssa_cache_evict(k, k.clone(), lens, torch.zeros(2, 2, 64), 10)
    with pytest.raises(ValueError):
        ssa_cache_accept(k, k.clone(), lens, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2), 5)


def test_tree_mask_from_parents():
    from SSA import tree_mask_from_parents

    mask = tree_mask_from_parents([-1, 0, 0, 2, -1, 4])
    want = torch.tensor([[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 0, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0],
                         [0, 0, 0, 0, 1, 0], [0, 0, 0, 0, 1, 1]], dtype=torch.bool)
    assert torch.equal(mask, want)
    both = tree_mask_from_parents([[-1, 0, 1], [-1, -1, -7]])
    assert torch.equal(both[0], torch.ones(3, 3).tril().bool()) and torch.equal(both[1], torch.eye(3).bool())
    for bad in ([0], [-1, 1], [[-1, 2, 0]], [-1.0, 0.0], [], [[[-1]]]):
        with pytest.raises(ValueError):
            tree_mask_from_parents(bad)


def test_native_functions_decline_host_tensors():
    nat = _lib.native()
    k, q, w = _cpu(1, 2, 64, 64), _cpu(1, 2, 3, 64), torch.zeros(1, 2, 64)
    lens, n = torch.tensor([64], dtype=torch.int32), torch.tensor(1.5)
    mask = torch.ones(3, 3, dtype=torch.bool)
    assert nat.tree(q, k, k, lens, mask, 0.1, n, n, 0, True, 0, 0) is None and nat.tree() is None
    assert nat.key_weights(q, k, w, lens, w, 0.1, n, n, 0, 0) is None and nat.key_weights(1) is None
    assert nat.evict(k, k, lens, w, 10, 0, 0, 0, 0) is None and nat.evict(None) is None
    assert nat.accept(k, k, lens, lens, lens, 3, 0, 0) is None and nat.accept() is None
    with pytest.raises(TypeError):
        nat.bind_cache(1)
    with pytest.raises(ValueError):
        nat.bind_cache(*[0] * 6)


def test_lookup_draft():
    from SSA.ssa_decoder import lookup_draft

    tokens, parents = lookup_draft(2, 3)([[7, 8, 1, 2, 7, 8], [1, 2, 3], [5, 5, 5, 5], [9]])
    assert tokens == [[1, 2, 7], [], [5], []]
    assert parents == [[-1, 0, 1], [], [-1], []]


def test_drafted_tree():
    """Node 0 is the last token; drafts that are no trees, too long ones and tokens
    outside the vocabulary (whose embedding would be read past the table) are refused."""
    from SSA.ssa_decoder import drafted_tree

    texts = [[3, 1], [4]]
    nodes, parents, mask = drafted_tree(texts, [[5, 6, 7], torch.tensor([9])], [[-1, 0, -1], [-1]], 4, 10)
    assert nodes == [[1, 5, 6, 7], [4, 9, 0, 0]] and parents == [[-1, 0, 1, 0], [-1, 0, 0, 0]]
    assert mask[0].tolist() == [[True, False, False, False], [True, True, False, False], [True, True, True, False],
                                [True, False, False, True]]
    assert drafted_tree(texts, [[], []], [[], []], 1, 10)[0] == [[1], [4]]
    for bad in (([[10], []], [[-1], []]), ([[-1], []], [[-1], []]), ([[1, 2, 3, 4], []], [[-1, 0, 1, 2], []]),
                ([[1], []], [[], []]), ([[1], []], [[0], []]), ([[1], []], [[-2], []]), ([[1]], [[-1]]),
                ([[1, 2], []], [[-1, 1], []])):
        with pytest.raises(ValueError):
            drafted_tree(texts, *bad, 4, 10)


def test_generate_refuses_budgets_that_cannot_hold():
    from SSA.ssa_decoder import SSADecoder, SSADecoderConfig

    model = SSADecoder(SSADecoderConfig(num_layers=1, hidden_size=64, num_attention_heads=1, num_query_groups=1,
                                        kv_channels=64, ffn_hidden_size=64, vocab_size=64))
    ids = torch.zeros(1, 4, dtype=torch.long)
    for bad in (dict(keep=0), dict(keep=10, sinks=8, recent=4), dict(keep=10, sinks=-1), dict(keep=64, slack=0)):
        with pytest.raises(ValueError):
            model.generate(ids, 2, **bad)
    with pytest.raises(ValueError):
        model.generate_drafted(ids, 2, None, max_nodes=2000)
    with pytest.raises(ValueError):
        model(ids, positions=torch.zeros(4, dtype=torch.long))
