"""Generation with drafted trees and bounded caches: the module's and the
decoder's paths through the cache operators."""

from __future__ import annotations

import math
import sys

import pytest
import torch

import cache_ops_ref as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _say(label):
    print(f"[gpu case] {label}", file=sys.stderr, flush=True)


def _qkv(dev, T, B, Hq, Hk, D, seed):
    g = torch.Generator().manual_seed(seed)
    return tuple((torch.randn(T, B, h, D, generator=g) * 0.5).to(BF16).to(dev) for h in (Hq, Hk, Hk))


def test_tree_step_is_the_branches_step_by_step(gpu):
    """Every node's context equals one decode step after another along its branch."""
    from SSA import SSAAttention, SSAKVCache, tree_mask_from_parents

    _say("tree step against decode steps")
    B, Hq, Hk, D, P = 2, 8, 2, 64, 50
    parents = [-1, 0, 0, 1, 2, 4]
    mod = SSAAttention(Hq, Hk, D).to(gpu).eval()
    qp, kp, vp = _qkv(gpu, P, B, Hq, Hk, D, 1)
    q, k, v = _qkv(gpu, len(parents), B, Hq, Hk, D, 2)
    with torch.no_grad():
        cache = SSAKVCache(B, Hk, 128, D, BF16, gpu)
        mod.forward_prompt(qp, kp, vp, cache)
        got = mod.forward_tree(q, k, v, cache, tree_mask_from_parents(parents).to(gpu))
        assert got.shape == (len(parents), B, Hq * D) and cache.seqlens.tolist() == [P + len(parents)] * B
        for node in range(len(parents)):
            branch, at = [], node
            while at >= 0:
                branch.insert(0, at)
                at = parents[at]
            one = SSAKVCache(B, Hk, 128, D, BF16, gpu)
            mod.forward_prompt(qp, kp, vp, one)
            for i in branch:
                want = mod.forward_decode(q[i:i + 1], k[i:i + 1], v[i:i + 1], one)
            # two kernels, each within two half steps of bf16 of the same value (below 1 here)
            assert (got[node].float() - want[0].float()).abs().max().item() <= 4 * 2.0 ** -8


def test_accepted_path_is_the_cache_of_its_tokens(gpu):
    """After accept, cache and weights are those of the accepted tokens one by one."""
    from SSA import SSAAttention, SSAKVCache, tree_mask_from_parents

    _say("accepted path")
    B, Hq, Hk, D, P = 3, 4, 2, 64, 40
    parents = [-1, 0, 0, 1, 2, 4, 5]
    mod = SSAAttention(Hq, Hk, D).to(gpu).eval()
    qp, kp, vp = _qkv(gpu, P, B, Hq, Hk, D, 3)
    q, k, v = _qkv(gpu, len(parents), B, Hq, Hk, D, 4)
    paths = [[0, 2, 4, 5], [0, 1, 3, 0], [0, 0, 0, 0]]
    counts = [4, 3, 0]
    with torch.no_grad():
        cache = SSAKVCache(B, Hk, 64, D, BF16, gpu, track_weights=True)
        mod.forward_prompt(qp, kp, vp, cache, window=8)
        before = cache.weights.clone()
        mod.forward_tree(q, k, v, cache, tree_mask_from_parents(parents).to(gpu))
        assert torch.equal(cache.weights, before)
        cache.accept(torch.tensor(paths), torch.tensor(counts), len(parents))
        assert cache.seqlens.tolist() == [P + c for c in counts]
        for b in range(B):
            one = SSAKVCache(1, Hk, 64, D, BF16, gpu, track_weights=True)
            mod.forward_prompt(qp[:, b:b + 1], kp[:, b:b + 1], vp[:, b:b + 1], one, window=8)
            for i in paths[b][:counts[b]]:
                mod.forward_decode(*(t[i:i + 1, b:b + 1] for t in (q, k, v)), one)
            L = P + counts[b]
            assert torch.equal(cache.k[b, :, :L], one.k[0, :, :L]) and torch.equal(cache.v[b, :, :L], one.v[0, :, :L])
            # normalisers of two kernels, each within 2^-16 (log2 units); 4 + 8 queries of 2 heads a group
            assert (cache.weights[b] - one.weights[0]).abs().max().item() <= 24 * 2.0 ** -15
            assert bool((cache.weights[b, :, L:] == 0).all())
    with pytest.raises(ValueError, match="nodes"):
        mod.forward_tree(q, k, v, cache, tree_mask_from_parents(parents).to(gpu))
        cache.accept(torch.tensor(paths), torch.tensor(counts), len(parents) - 1)


def test_weights_of_a_generation_add_up(gpu):
    """Every query's probabilities add up to 1 over the cache."""
    from SSA import SSAAttention, SSAKVCache

    _say("weights add up")
    B, Hq, Hk, D, P, new = 2, 8, 4, 64, 100, 5
    mod = SSAAttention(Hq, Hk, D).to(gpu).eval()
    q, k, v = _qkv(gpu, P + new, B, Hq, Hk, D, 5)
    cache = SSAKVCache(B, Hk, 160, D, BF16, gpu, track_weights=True)
    with torch.no_grad():
        mod.forward_prompt(q[:P], k[:P], v[:P], cache, window=16)
        for t in range(P, P + new):
            mod.forward_decode(q[t:t + 1], k[t:t + 1], v[t:t + 1], cache)
    total = cache.weights.sum(-1)
    want = float((16 + new) * (Hq // Hk))
    assert torch.allclose(total, torch.full_like(total, want), rtol=2.0 ** -12)
    before = cache.weights.clone()
    kept = cache.evict(40, sinks=2, recent=8)
    assert cache.seqlens.tolist() == [40] * B and kept.shape == (B, Hk, 40)
    _, left, rows = ref.evict([P + new] * B, before, 40, 2, 8)
    assert torch.equal(kept.cpu(), rows) and torch.equal(cache.weights.cpu(), left)


def test_caches_without_weights_refuse(gpu):
    from SSA import SSAKVCache

    cache = SSAKVCache(1, 2, 64, 64, BF16, gpu)
    with pytest.raises(ValueError, match="track"):
        cache.evict(10)
    with pytest.raises(ValueError, match="track"):
        cache.add_weights(torch.zeros(1, 2, 64, dtype=BF16, device=gpu), torch.zeros(1, 2, device=gpu), 0.1, 1.5, 0.8)


def test_refusals_on_the_gpu(gpu):
    """What the operators cannot take raises, in both launch paths."""
    from SSA import ssa_cache_accept, ssa_cache_evict, ssa_key_weights, ssa_tree_attention

    _say("refusals")
    k = torch.zeros(2, 2, 64, 64, dtype=BF16, device=gpu)
    v, q = torch.zeros_like(k), torch.zeros(2, 4, 5, 64, dtype=BF16, device=gpu)
    lens = torch.tensor([64, 10], dtype=torch.int32, device=gpu)
    mask = torch.ones(5, 5, dtype=torch.bool, device=gpu)
    w, m = torch.zeros(2, 2, 64, device=gpu), torch.zeros(2, 4, 5, device=gpu)
    tree = lambda q=q, k=k, v=v, lens=lens, mask=mask: ssa_tree_attention(q, k, v, lens, mask, 0.1, 1.5, 0.8)  # noqa: E731
    for bad in (dict(mask=mask[:4]), dict(mask=mask[None]), dict(lens=lens[:1]), dict(lens=lens.float()),
                dict(q=q.half()), dict(q=q[:1]), dict(q=q[..., :32]), dict(k=k[:, :1]), dict(v=v.half()),
                dict(k=k.transpose(2, 3)), dict(q=torch.zeros(2, 4, 1025, 64, dtype=BF16, device=gpu))):
        with pytest.raises(ValueError):
            tree(**bad)
    with pytest.raises(AssertionError):
        tree(q=torch.zeros(2, 3, 5, 64, dtype=BF16, device=gpu))
    add = lambda q=q, m=m, w=w: ssa_key_weights(q, k, m, lens, w, 0.1, 1.5, 0.8)  # noqa: E731
    for bad in (dict(m=m[..., :4]), dict(w=w.half()), dict(w=w[:, :1]), dict(w=torch.zeros(2, 2, 128, device=gpu)[..., ::2]),
                dict(w=torch.zeros(2, 1, 64, device=gpu).expand(2, 2, 64)), dict(m=m.cpu()),
                dict(q=torch.zeros(2, 4, 65, 64, dtype=BF16, device=gpu), m=torch.zeros(2, 4, 65, device=gpu))):
        with pytest.raises(ValueError):
            add(**bad)
    cut = lambda k=k, v=v, w=w, keep=10, **kw: ssa_cache_evict(k, v, lens, w, keep, **kw)  # noqa: E731
    for bad in (dict(keep=0), dict(keep=65), dict(sinks=6, recent=5), dict(sinks=-1), dict(v=k),
                dict(k=k[:, :1].expand(2, 2, 64, 64)), dict(w=w[..., :32])):
        with pytest.raises(ValueError):
            cut(**bad)
    path, n = torch.zeros(2, 3, dtype=torch.int32, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    take = lambda k=k, v=v, path=path, n=n, nodes=5: ssa_cache_accept(k, v, lens, path, n, nodes)  # noqa: E731
    for bad in (dict(nodes=2), dict(nodes=0), dict(nodes=1025), dict(path=path[:1]), dict(path=path[:, :0]),
                dict(n=n[:1]), dict(v=k), dict(v=v[:, :1].expand(2, 2, 64, 64)), dict(path=path.float())):
        with pytest.raises(ValueError):
            take(**bad)
    assert bool((k == 0).all()) and bool((w == 0).all())


# ------------------------------------------------------------------ the decoder
def test_accept_of_another_tree_leaves_the_cache(gpu):
    """A number of nodes that is not the last tree's is refused before anything moves."""
    from SSA import SSAAttention, SSAKVCache

    _say("accept with another number of nodes")
    mod = SSAAttention(4, 2, 64).to(gpu).eval()
    cache = SSAKVCache(1, 2, 64, 64, BF16, gpu, track_weights=True)
    with torch.no_grad():
        mod.forward_prompt(*_qkv(gpu, 20, 1, 4, 2, 64, 3), cache)
        mod.forward_tree(*_qkv(gpu, 5, 1, 4, 2, 64, 4), cache, torch.ones(5, 5, device=gpu).tril())
    before = [t.clone() for t in (cache.k, cache.v, cache.seqlens, cache.weights)]
    with pytest.raises(ValueError):
        cache.accept(torch.tensor([[0, 2]], device=gpu), torch.tensor([2], device=gpu), 6)
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.seqlens, cache.weights)))
    with pytest.raises(ValueError):
        cache.accept(torch.tensor([[0.0, 2.5]], device=gpu), torch.tensor([2], device=gpu), 5)
    cache.accept(torch.tensor([[0, 2]], device=gpu), torch.tensor([2], device=gpu), 5)
    assert cache.seqlens.tolist() == [22]
    # 4 heads, 22 tokens, at most 1 each: node 2 also paid node 1, which did not stay
    # (the normalisers are fp32 sums, each p within 2^-12 of its own)
    assert float(cache.weights.sum()) <= 4 * 22 * (1 + 2.0 ** -12)


def _decoder(gpu, **kw):
    from SSA.ssa_decoder import SSADecoder, SSADecoderConfig

    torch.manual_seed(0)
    cfg = SSADecoderConfig(num_layers=2, hidden_size=256, num_attention_heads=4, num_query_groups=2, kv_channels=64,
                           ffn_hidden_size=512, vocab_size=512, init_std=0.1, **kw)
    return SSADecoder(cfg).to(gpu).eval()


def _picks_are_the_models(model, tokens, P):
    """Every token after the prompt has the largest logit of the dense forward over
    the text before it, within the logits' bf16 rounding through the layers."""
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        logits = model(tokens[:, :-1])[P - 1:].float()  # [new, B, V]
    best = logits.max(-1).values
    got = logits.gather(-1, tokens[:, P:].t()[..., None])[..., 0]
    scale = logits.abs().amax(-1)
    assert bool((best - got <= 2.0 ** -4 * scale).all()), float((best - got).max())


@pytest.mark.parametrize("B", [1, 3])
def test_generate_drafted_gives_the_models_picks(gpu, B):
    from SSA.ssa_decoder import lookup_draft

    _say(f"generate_drafted B={B}")
    model = _decoder(gpu)
    ids = torch.randint(512, (B, 20), generator=torch.Generator().manual_seed(1)).to(gpu)
    plain, _ = model.generate(ids, 24)
    _picks_are_the_models(model, plain, 20)
    tokens, steps = model.generate_drafted(ids, 24, lookup_draft(1, 5))
    assert tokens.shape == (B, 44) and torch.equal(tokens[:, :20], ids) and 1 <= steps <= 23
    _picks_are_the_models(model, tokens, 20)

    # a draft that knows the answer: a wrong sibling before every right token
    def known(texts):
        drafted, above = [], []
        for seq, want in zip(texts, plain.tolist()):
            right = want[len(seq):len(seq) + 4] if seq == want[:len(seq)] else []
            toks, par, at = [], [], -1
            for t in right:
                toks += [(t + 1) % 512, t]
                par += [at, at]
                at = len(toks) - 1
            drafted.append(toks)
            above.append(par)
        return drafted, above

    tokens, fewer = model.generate_drafted(ids, 24, known)
    _picks_are_the_models(model, tokens, 20)
    # five tokens a step where the tree's and the decode step's picks agree throughout
    if torch.equal(tokens, plain):
        assert fewer <= 5
    with pytest.raises(ValueError):
        model.generate_drafted(ids, 4, lambda texts: ([[1] * 100] * B, [[-1] * 100] * B))
    with pytest.raises(ValueError):
        model.generate_drafted(ids, 4, lambda texts: ([[1, 2]] * B, [[1, -1]] * B))


def test_generate_with_a_budget(gpu):
    """A budget that holds everything changes no token; a smaller one bounds every
    cache and generates on."""
    _say("generate with a budget")
    model = _decoder(gpu)
    ids = torch.randint(512, (2, 40), generator=torch.Generator().manual_seed(2)).to(gpu)
    plain, logits = model.generate(ids, 30)
    whole, same = model.generate(ids, 30, keep=100)
    # prompt and decode kernels are the same; only the returned normaliser differs
    assert torch.equal(plain, whole) and torch.equal(logits, same)
    held = []
    make = model.new_caches

    def spy(*args, **kw):
        held.extend(make(*args, **kw))
        return held

    model.new_caches = spy
    tokens, steps = model.generate(ids, 30, keep=24, sinks=2, recent=8, slack=6)
    assert tokens.shape == (2, 70) and bool(steps.isfinite().all())
    for cache in held:
        assert cache.capacity == 40 and bool((cache.seqlens <= 30).all()) and bool((cache.weights >= 0).all())
        assert bool((cache.weights[..., 31:] == 0).all())


def test_positions_of_their_own(gpu):
    """positions [B, S] equal the shared ones where they are the same."""
    _say("positions")
    for fused in (True, False):
        model = _decoder(gpu, fused_rope=fused)
        ids = torch.randint(512, (3, 17), generator=torch.Generator().manual_seed(3)).to(gpu)
        with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
            a = model(ids, start_pos=5)
            b = model(ids, positions=torch.arange(5, 22, device=gpu).expand(3, 17))
        assert torch.equal(a, b)


def test_drafted_generation_in_fp16_and_head_dim_128(gpu):
    from SSA.ssa_decoder import SSADecoder, SSADecoderConfig, lookup_draft

    _say("fp16 head dim 128")
    torch.manual_seed(1)
    model = SSADecoder(SSADecoderConfig(num_layers=1, hidden_size=256, num_attention_heads=2, num_query_groups=1,
                                        kv_channels=128, ffn_hidden_size=256, vocab_size=256, init_std=0.1))
    model = model.to(gpu).eval()
    ids = torch.randint(256, (2, 9), generator=torch.Generator().manual_seed(4)).to(gpu)
    tokens, _ = model.generate_drafted(ids, 12, lookup_draft(1, 3), dtype=torch.float16)
    assert tokens.shape == (2, 21)
    out, _ = model.generate(ids, 12, dtype=torch.float16, keep=12, sinks=1, recent=4, slack=3)
    assert out.shape == (2, 21) and math.isfinite(float(out.float().mean()))
