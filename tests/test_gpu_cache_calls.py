"""Calls of the cached-generation paths on the GPU that must be refused, or leave
things as they are."""

from __future__ import annotations

import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _say(label):
    print(f"[gpu case] {label}", file=sys.stderr, flush=True)


def _step(dev, T, B, Hq, Hk, D, seed, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(T, B, h, D, generator=g).to(dtype).to(dev) for h in (Hq, Hk, Hk))


def _held(cache):
    return [t.clone() for t in (cache.k, cache.v, cache.seqlens, *([] if cache.weights is None else [cache.weights]))]


def test_refused_trees_leave_the_cache(gpu):
    from SSA import SSAAttention, SSAKVCache

    _say("refused trees")
    mod = SSAAttention(4, 2, 64).to(gpu).eval()
    cache = SSAKVCache(2, 2, 32, 64, BF16, gpu)
    mod.forward_prompt(*_step(gpu, 10, 2, 4, 2, 64, 1), cache)
    before = _held(cache)
    for T, mask, dtype in ((5, (4, 5), BF16), (5, (3, 5, 5), BF16), (33, (33, 33), BF16), (5, (5, 5), torch.float16)):
        with pytest.raises(ValueError):
            mod.forward_tree(*_step(gpu, T, 2, 4, 2, 64, 2, dtype), cache, torch.ones(mask, device=gpu))
        assert all(torch.equal(a, b) for a, b in zip(before, _held(cache)))
    q, k, v = _step(gpu, 5, 2, 4, 2, 64, 3)
    want = mod.forward_tree(q, k, v, cache, torch.ones(5, 5).tril())
    assert cache.seqlens.tolist() == [15, 15]
    # again with gradients on and a mask that the device holds
    cache.seqlens -= 5
    got = mod.forward_tree(q.requires_grad_(), k.requires_grad_(), v, cache, torch.ones(5, 5, device=gpu).tril())
    assert torch.equal(got, want) and not got.requires_grad and not cache.k.requires_grad


@pytest.mark.parametrize("layout", ["row", "token", "head", "slots"])
def test_one_buffer_of_keys_and_values(gpu, layout):
    """Keys and values side by side in one buffer share no element and are moved as
    two buffers are; views that share some are refused and nothing moves."""
    from SSA import ssa_cache_accept, ssa_cache_evict

    _say(f"one buffer, by {layout}")
    B, H, cap, D = 3, 2, 200, 64
    g = torch.Generator().manual_seed(2)
    make = lambda *shape: torch.randn(*shape, generator=g).to(BF16).to(gpu)  # noqa: E731
    if layout == "row":
        room = make(B, H, cap, 2 * D)
        k, v, wrong = room[..., :D], room[..., D:], room[..., D // 2:D // 2 + D]
    elif layout == "token":
        room = make(B, cap, 2, H, D)
        k, v, wrong = room[:, :, 0].transpose(1, 2), room[:, :, 1].transpose(1, 2), room[:, :, :, 0].transpose(1, 2)
    elif layout == "head":
        room = make(B, H, 2 * cap, D)
        k, v, wrong = room[:, :, :cap], room[:, :, cap:], room[:, :, 5:cap + 5]
    else:  # keys in slots 0, 2, 4 and values in 3, 5, 7
        room = make(8, H, cap, D)
        k, v, wrong = room[0:6:2], room[3:8:2], room[2:8:2]
    kc, vc = k.clone(), v.clone()
    lens = torch.tensor([200, 150, 40], dtype=torch.int32, device=gpu)
    w = torch.rand(B, H, cap, generator=g).to(gpu)
    path = torch.tensor([[1, 4, 9], [0, 2, 3], [5, 6, 7]], dtype=torch.int32, device=gpu)
    count = torch.tensor([3, 2, 1], dtype=torch.int32, device=gpu)
    before = room.clone()
    for a, b in ((k, wrong), (wrong, k)):
        with pytest.raises(ValueError):
            ssa_cache_accept(a, b, lens, path, count, 10)
        with pytest.raises(ValueError):
            ssa_cache_evict(a, b, lens, w, 60)
    torch.cuda.synchronize()
    assert torch.equal(room, before)
    one, two = ssa_cache_accept(k, v, lens, path, count, 10), ssa_cache_accept(kc, vc, lens, path, count, 10)
    assert torch.equal(one, two) and torch.equal(k, kc) and torch.equal(v, vc)
    one, two = ssa_cache_evict(k, v, lens, w, 60, 2, 8), ssa_cache_evict(kc, vc, lens, w, 60, 2, 8)
    assert all(torch.equal(x, y) for x, y in zip(one, two)) and torch.equal(k, kc) and torch.equal(v, vc)
    ssa_cache_evict(v, k, lens, w, 60)  # either of them first


def test_a_token_drafted_twice_does_not_end_the_path(gpu):
    """Siblings with one token, the first of which nothing follows: the path goes on
    through the other one, four drafted tokens a step."""
    from SSA.ssa_decoder import SSADecoder, SSADecoderConfig

    _say("a token drafted twice")
    torch.manual_seed(0)
    model = SSADecoder(SSADecoderConfig(num_layers=2, hidden_size=256, num_attention_heads=4, num_query_groups=2,
                                        kv_channels=64, ffn_hidden_size=512, vocab_size=512, init_std=0.1))
    model = model.to(gpu).eval()
    ids = torch.randint(512, (2, 20), generator=torch.Generator().manual_seed(1)).to(gpu)
    plain, _ = model.generate(ids, 24)

    def twice(texts):
        drafted, above = [], []
        for seq, want in zip(texts, plain.tolist()):
            tokens, parents, at = [], [], -1
            for t in want[len(seq):len(seq) + 4] if seq == want[:len(seq)] else []:
                tokens += [t, t]
                parents += [at, at]
                at = len(tokens) - 1
            drafted.append(tokens)
            above.append(parents)
        return drafted, above

    tokens, steps = model.generate_drafted(ids, 24, twice)
    # five tokens a step where the tree's and the decode step's picks agree throughout
    if torch.equal(tokens, plain):
        assert steps <= 5
