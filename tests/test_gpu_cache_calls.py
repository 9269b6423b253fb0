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
