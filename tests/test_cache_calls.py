"""Calls of the cached-generation paths that must be refused, or leave things as
they are, without a GPU."""

from __future__ import annotations

import pytest
import torch


def _model():
    from SSA.ssa_decoder import SSADecoder, SSADecoderConfig

    return SSADecoder(SSADecoderConfig(num_layers=1, hidden_size=64, num_attention_heads=1, num_query_groups=1,
                                       kv_channels=64, ffn_hidden_size=64, vocab_size=64))


def test_a_tree_needs_caches():
    """A tree's mask without caches would be the plain causal forward's, unseen."""
    model = _model()
    ids, mask = torch.zeros(2, 4, dtype=torch.long), torch.eye(4, dtype=torch.bool)
    with pytest.raises(ValueError, match="caches"):
        model(ids, tree_mask=mask)
    with pytest.raises(ValueError, match="caches"):
        model(ids, positions=torch.zeros(2, 4, dtype=torch.long), tree_mask=mask)
    layer = model.layers[0]
    x = torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="cache"):
        layer.self_attention(x, model.rotary(torch.arange(4)), None, mask)


def _module_on_host(monkeypatch):
    """An SSAAttention whose tree attention is a stand-in that runs on the host."""
    import SSA.ssa_attention as module

    def attention(q, k_cache, v_cache, lens, mask, scale, n, b, num_splits=0, return_m=False):
        out = q.detach().clone()
        return (out, torch.zeros(q.shape[:3])) if return_m else out

    monkeypatch.setattr(module, "ssa_tree_attention", attention)
    monkeypatch.setattr(module, "check_tree_call", lambda *args: None, raising=False)
    return module.SSAAttention(2, 1, 64)


@pytest.mark.parametrize("track", [False, True])
def test_appends_hang_no_graph_on_the_cache(monkeypatch, track):
    """Keys and values that need gradients leave none in the cache's buffers, and a
    tree's queries, kept for its accepted path, hold no graph alive."""
    from SSA import SSAKVCache

    mod = _module_on_host(monkeypatch)
    cache = SSAKVCache(2, 1, 16, 64, torch.bfloat16, "cpu", track_weights=track)
    make = lambda T, H: torch.ones(T, 2, H, 64, dtype=torch.bfloat16, requires_grad=True) * 2  # noqa: E731
    k, v = make(3, 1), make(3, 1)
    cache.append(k.permute(1, 2, 0, 3), v.permute(1, 2, 0, 3))
    assert not cache.k.requires_grad and not cache.v.requires_grad and cache.seqlens.tolist() == [3, 3]
    assert bool((cache.k[:, :, :3] == 2).all()) and bool((cache.v[:, :, 3:] == 0).all())
    q = make(4, 2)
    ctx = mod.forward_tree(q, make(4, 1), make(4, 1), cache, torch.ones(4, 4).tril())
    assert not cache.k.requires_grad and not cache.v.requires_grad and not ctx.requires_grad
    if track:
        kept = cache._drafted[0]
        assert not kept.requires_grad and (kept._base is None or kept._base.grad_fn is None)


def test_a_refused_tree_leaves_the_cache(monkeypatch):
    """forward_tree raises before anything is appended."""
    from SSA import SSAAttention, SSAKVCache

    mod = SSAAttention(2, 1, 64)
    cache = SSAKVCache(2, 1, 16, 64, torch.bfloat16, "cpu")  # on the host: refused
    make = lambda T, H: torch.ones(T, 2, H, 64, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError):
        mod.forward_tree(make(4, 2), make(4, 1), make(4, 1), cache, torch.ones(4, 4).tril())
    assert cache.seqlens.tolist() == [0, 0] and bool((cache.k == 0).all())


@pytest.mark.parametrize("T,mask,dtype,D", [
    (4, (4, 3), torch.bfloat16, 64), (4, (3, 4, 4), torch.bfloat16, 64), (1025, (1025, 1025), torch.bfloat16, 64),
    (17, (17, 17), torch.bfloat16, 64), (4, (4, 4), torch.float32, 64), (4, (4, 4), torch.float16, 64),
    (4, (4, 4), torch.bfloat16, 256)])
def test_what_a_tree_call_refuses(monkeypatch, T, mask, dtype, D):
    """The checks that forward_tree makes before it appends, on tensors that say they
    are on the GPU."""
    import SSA.ssa_cache_ops as ops
    from SSA import SSAAttention, SSAKVCache

    monkeypatch.setattr(ops, "_on_gpu", lambda t: True, raising=False)
    mod = SSAAttention(2, 1, D)
    cache = SSAKVCache(2, 1, 16, D, torch.bfloat16, "cpu")
    make = lambda H: torch.ones(T, 2, H, D, dtype=dtype)  # noqa: E731
    with pytest.raises(ValueError) as why:
        mod.forward_tree(make(2), make(1), make(1), cache, torch.ones(mask))
    assert "GPU" not in str(why.value)
    assert cache.seqlens.tolist() == [0, 0] and bool((cache.k == 0).all())


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.int16, torch.uint8, torch.bool])
def test_accepted_counts_of_any_integer_type(monkeypatch, dtype):
    """A tracking cache takes what ssa_cache_accept takes: with counts of 8 bits
    it raised after the rows had moved, for 300 nodes do not fit them."""
    import SSA.ssa_attention as module
    from SSA import SSAKVCache

    mod = _module_on_host(monkeypatch)
    nodes, seen = 300, {}
    cache = SSAKVCache(2, 1, 512, 64, torch.bfloat16, "cpu", track_weights=True)
    make = lambda T, H: torch.ones(T, 2, H, 64, dtype=torch.bfloat16)  # noqa: E731
    mod.forward_tree(make(nodes, 2), make(nodes, 1), make(nodes, 1), cache, torch.ones(nodes, nodes).tril())

    def accept(k, v, lens, path, accepted, n):
        return (lens - n + accepted.to(torch.int32).clamp(0, path.shape[1])).int()

    def weights(q, k, m, lens, w, *rest):
        seen.update(m=m, lens=lens.tolist())

    monkeypatch.setattr(module, "ssa_cache_accept", accept)
    monkeypatch.setattr(module, "ssa_key_weights", weights)
    path = torch.arange(nodes).expand(2, nodes)
    cache.accept(path, torch.tensor([1, 0]).to(dtype), nodes)
    assert cache.seqlens.tolist() == [1, 0] and seen["lens"] == [1, 0]
    # one query counts for the first sequence, none for the second
    assert (seen["m"] > -torch.inf).sum((1, 2)).tolist() == [2, 0]


def test_nothing_is_accepted_of_more_nodes_than_rows(monkeypatch):
    """Lengths past the capacity hold as many rows as there are: of a tree of more
    nodes than that nothing is accepted, and no weights are added."""
    import SSA.ssa_attention as module
    from SSA import SSAKVCache

    cache = SSAKVCache(1, 1, 8, 64, torch.bfloat16, "cpu", track_weights=True)
    cache.seqlens += 20
    cache._drafted = (torch.zeros(1, 2, 12, 64), torch.zeros(1, 2, 12), 0.1, 1.5, 0.8)
    seen = []
    monkeypatch.setattr(module, "ssa_cache_accept", lambda k, v, lens, *rest: lens.clamp(max=8))
    monkeypatch.setattr(module, "ssa_key_weights", lambda q, k, m, *rest: seen.append(m))
    cache.accept(torch.arange(3)[None], torch.tensor([3]), 12)
    assert cache.seqlens.tolist() == [8] and all(bool((m == -torch.inf).all()) for m in seen)


CACHE_BYTES = 2 * 4 * 8 * 4096 * 64  # of the caches below


@pytest.mark.parametrize("entry", ["ssa_cache_evict", "ssa_cache_accept"])
@pytest.mark.parametrize("offset,strides", [
    (16, None), (64, None), (128 * 100, None), (CACHE_BYTES - 128, None), (-128, None), (-CACHE_BYTES + 128, None),
    (4096 * 128, None),                               # a head further
    (64, (8 * 4096 * 128, 4096 * 128, 128)),          # rows that reach into each other's half
    (192, (8 * 4096 * 128, 4096 * 128, 128)),
    (2 * 64 * 4096, (8 * 4096 * 64, 64, 8 * 64)),     # another layout over the same bytes
])
def test_caches_that_overlap_are_refused(entry, offset, strides):
    """Keys and values that share memory would be moved over each other."""
    import ctypes

    from SSA import _lib

    base = 1 << 32
    k = _lib.Tensor4(base, *((8 * 4096 * 64, 4096 * 64, 64) if strides is None or strides[2] == 512 else strides))
    v = _lib.Tensor4(base + offset, *(strides or (8 * 4096 * 64, 4096 * 64, 64)))
    far = 1 << 20
    if entry == "ssa_cache_evict":
        args = _lib.CacheEvictArgs(k, v, far, 8 * 4096, 4096, far, far + 64, far + 4096, far, 4, 8, 4096, 64,
                                   _lib.SSA_DTYPE_BF16, 1024, 4, 64)
    else:
        args = _lib.CacheAcceptArgs(k, v, far, far, far, far + 64, 4, 8, 4096, 64, _lib.SSA_DTYPE_BF16, 16, 5)
    assert getattr(_lib.lib(), entry)(ctypes.byref(args), None) == _lib.SSA_ERR_ALIGNMENT


def test_the_longest_drafted_path_is_kept():
    """Of siblings with one token the one that leads furthest; a path ends where the
    model's pick was not drafted, or after `most` tokens."""
    from SSA.ssa_decoder import longest_path

    #        0
    #     1     2     3      nodes 1 and 3 hold the token that the model picks
    #           4     5 - 6
    tokens, parents = [9, 7, 8, 7, 5, 4, 3], [-1, 0, 0, 0, 2, 3, 5]
    picks = [7, 4, 5, 4, 1, 3, 2]
    assert longest_path(tokens, parents, picks, 10) == [0, 3, 5, 6]
    assert longest_path(tokens, parents, picks, 3) == [0, 3, 5]
    assert longest_path(tokens, parents, picks, 1) == [0]
    assert longest_path(tokens, parents, [8, 0, 5, 0, 1, 0, 0], 10) == [0, 2, 4]
    assert longest_path(tokens, parents, [6] * 7, 10) == [0]
    # of equally long ones the first
    assert longest_path([9, 7, 7], [-1, 0, 0], [7, 1, 1], 10) == [0, 1]
    # nodes that only fill a shorter draft up are no drafted tokens
    assert longest_path([9, 0, 0], [-1, 0, 0], [0, 0, 0], 10, drafted=0) == [0]


def test_a_prompt_longer_than_its_cache_is_refused(monkeypatch):
    """Before anything is computed or appended; one that fills the cache is taken."""
    import SSA.ssa_attention as module
    from SSA import SSAKVCache

    monkeypatch.setattr(module, "ssa_flash_attn_forward",
                        lambda q, k, v, *rest: (torch.zeros_like(q), torch.zeros(q.shape[:3])))
    mod = module.SSAAttention(2, 1, 64)
    cache = SSAKVCache(1, 1, 8, 64, torch.bfloat16, "cpu")
    make = lambda T, H: torch.ones(T, 1, H, 64, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError, match="rows"):
        mod.forward_prompt(make(9, 2), make(9, 1), make(9, 1), cache)
    assert cache.seqlens.tolist() == [0] and bool((cache.k == 0).all())
    mod.forward_prompt(make(8, 2), make(8, 1), make(8, 1), cache)
    assert cache.seqlens.tolist() == [8]


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 256), (torch.float16, 16)])
def test_a_cache_tracks_what_the_operators_take(dtype, D):
    """A cache whose weights no operator can add to is refused when it is made, not
    at its first step, with the step's rows already in it."""
    from SSA import SSAKVCache
    from SSA.ssa_decoder import SSADecoder, SSADecoderConfig

    assert SSAKVCache(1, 1, 8, D, dtype, "cpu").weights is None
    with pytest.raises(ValueError):
        SSAKVCache(1, 1, 8, D, dtype, "cpu", track_weights=True)
    model = SSADecoder(SSADecoderConfig(num_layers=1, hidden_size=D, num_attention_heads=1, num_query_groups=1,
                                        kv_channels=D, ffn_hidden_size=64, vocab_size=64))
    with pytest.raises(ValueError, match="weights"):
        model.generate(torch.zeros(1, 4, dtype=torch.long), 2, dtype=dtype, keep=100)


def test_a_prompt_whose_attention_cannot_be_weighed_is_refused(monkeypatch):
    """Queries of another type than a tracking cache's: before anything is appended."""
    import SSA.ssa_attention as module
    from SSA import SSAKVCache

    monkeypatch.setattr(module, "ssa_flash_attn_forward",
                        lambda q, k, v, *rest: (torch.zeros_like(q), torch.zeros(q.shape[:3])))
    mod = module.SSAAttention(2, 1, 64)
    make = lambda H: torch.ones(4, 1, H, 64, dtype=torch.float16)  # noqa: E731
    cache = SSAKVCache(1, 1, 8, 64, torch.bfloat16, "cpu", track_weights=True)
    with pytest.raises(ValueError):
        mod.forward_prompt(make(2), make(1), make(1), cache)
    assert cache.seqlens.tolist() == [0] and bool((cache.k == 0).all())
    mod.forward_prompt(make(2), make(1), make(1), cache, window=0)  # nothing to weigh
    assert cache.seqlens.tolist() == [4]
