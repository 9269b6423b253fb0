"""Tree attention over long caches whose keys' probabilities are tiny beside the
largest: in fp16 they are subnormal, and below 2^-25 nothing, so the kernel keeps
its exponents' reference 10 below the largest one.  Every key then counts within 2^-25
of a weight of at least 2^10, that is 2^-35 of its row's sum."""

from __future__ import annotations

import math
import sys

import pytest
import torch

import cache_ops_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
SUBNORMAL = 2.0 ** -35


def _say(label):
    print(f"[gpu case] {label}", file=sys.stderr, flush=True)


def _check(dev, q, k, v, mask, scale, n, b, splits):
    """Full caches: out within the definition's bound (cache_ops_ref) plus, in fp16, 2^-35 |v| of every key."""
    from SSA import ssa_tree_attention

    lens = [k.shape[2]] * k.shape[0]
    out, m = ssa_tree_attention(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), mask.to(dev), scale,
                                torch.tensor(n, device=dev), torch.tensor(b, device=dev), num_splits=splits,
                                return_m=True)
    torch.cuda.synchronize()
    want, wm, tol, mtol = ref.tree(q, k, v, lens, mask.to(dev), scale, n, b)
    if q.dtype == FP16:
        every = v.double().abs().sum(2).repeat_interleave(q.shape[1] // k.shape[1], 1)  # [B, Hq, D]
        tol = tol + SUBNORMAL * every[:, :, None, :]
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), f"out: error {float(off.max())}, {float((off - tol).max())} over its bound"
    assert bool(((m.double() - wm).abs() <= mtol).all())
    return want


# B, Hq, Hkv, capacity, T and the rows of a workgroup that the library's plan has for one split
FORMS = [((1, 1, 1, 1 << 16, 1), 32), ((1, 16, 1, 4096, 1024), 64), ((4, 64, 8, 4096, 65), 128),
         ((8, 64, 8, 4096, 65), 256)]


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("call", [c for c, _ in FORMS])
def test_many_keys_below_half_of_the_smallest(gpu, D, dtype, call):
    """A key of weight 2^25.06 in each of the first 16 tiles of 32 keys, with zeros for
    values, and else keys of weight 1: the result is theirs.  The T nodes see
    themselves only."""
    B, Hq, Hk, L, T = call
    _say(f"small weights D={D} {dtype} {call}")
    k = torch.zeros(B, Hk, L, D, dtype=dtype, device=gpu)
    v = torch.full((B, Hk, L, D), 1024.0, dtype=dtype, device=gpu)
    v[..., ::3] = -768.0
    q = torch.ones(B, Hq, T, D, dtype=dtype, device=gpu)
    k[:, :, 0:512:32] = 31.25  # scale q.k = 31.25: t = 5 log2(32.25) = 25.06
    v[:, :, 0:512:32] = 0.0
    want = _check(gpu, q, k, v, torch.eye(T, dtype=torch.bool), 1.0 / D, 5.0, 1.0, 1)
    assert bool((want[..., 1] > 1024 * 0.99 * (L - 16 - T) / (16 * 2.0 ** 25.06)).all())


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T,splits", [(3, 1), (3, 0), (40, 1), (40, 12)])
def test_spread_exponents_in_fp16(gpu, D, T, splits):
    """Random scores under n = 5 (exponents of -13 to 17 and more) and one dominant key."""
    _say(f"spread exponents D={D} T={T} splits={splits}")
    L = 20000
    g = torch.Generator().manual_seed(D + T)
    k = torch.randn(1, 2, L, D, generator=g).to(FP16).to(gpu)
    v = torch.randn(1, 2, L, D, generator=g).to(FP16).to(gpu)
    q = (2 * torch.randn(1, 4, T, D, generator=g)).to(FP16).to(gpu)
    k[:, :, 777] = 3 * q[:, ::2, 0]
    _check(gpu, q, k, v, torch.ones(T, T, dtype=torch.bool).tril(), 1.0 / math.sqrt(D), 5.0, 0.8, splits)


@pytest.mark.parametrize("n", [1.5, -5.0, 0.0, 5.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rising_and_falling_scores(gpu, n, dtype):
    """Scores that rise or fall along the cache move the reference on, or leave it behind."""
    _say(f"rising scores n={n} {dtype}")
    L, D, T = 4000, 64, 33
    g = torch.Generator().manual_seed(5)
    ramp = torch.linspace(-6, 6, L)[:, None] * torch.ones(D)
    v = torch.randn(1, 1, L, D, generator=g).to(dtype).to(gpu)
    q = (1 + 0.2 * torch.randn(1, 2, T, D, generator=g)).to(dtype).to(gpu)
    for keys in (ramp, ramp.flip(0)):
        k = keys[None, None].to(dtype).to(gpu).contiguous()
        _check(gpu, q, k, v, torch.ones(T, T, dtype=torch.bool).tril(), 0.125, n, 0.8, 1)
