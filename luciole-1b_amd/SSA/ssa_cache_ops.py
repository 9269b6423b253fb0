"""Operators on a KV cache for generation with drafted tokens and a bounded cache.

* ``ssa_tree_attention``: the tokens of a drafted tree attend the cached prefix
  and their own branch, in one pass over the cache;
* ``ssa_key_weights``: the attention that the last queries paid to every cached
  key is added to the keys' weights;
* ``ssa_cache_evict``: the cache is cut to the rows of largest weight;
* ``ssa_cache_accept``: the accepted path of a tree moves to the end of the prefix.

They stand beside ``ssa_decode_attention`` (``ssa_hip_kernel``) and take the
same caches: ``[B, Hkv, capacity, D]`` in bf16 or fp16, head dims 32, 64 and
128, any strides whose last one is 1, used in place; ``cache_seqlens`` holds
int32 lengths ``[B]``, read and clamped to ``[0, capacity]`` on the device, so
no call synchronises.  None has a gradient (generation only).  No reference
counterpart: the reference's generation loop re-runs the whole prefix per token
(training/train/train_ssa_triton/generate_triton.py:315-331).  The C entry
points are in include/ssa_cache_ops.h.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ssa_hip_kernel import (_DTYPES, _check_cache_layout, _current, _is_pow2, _kernel_layout, _native_result, _scalar,
                             _t4)

MAX_TREE_NODES = 1024
HEAD_DIMS = (32, 64, 128)


def _on_gpu(t) -> bool:
    return t.is_cuda


def _check_caches(k_cache, v_cache, names=("k_cache", "v_cache")):
    """Shapes, types, devices and layouts of a pair of caches."""
    for t, name in zip((k_cache, v_cache), names):
        if not torch.is_tensor(t) or t.dim() != 4:
            raise ValueError(f"{name} must be [B, Hkv, capacity, D]")
        if t.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"unsupported dtype {t.dtype}: the caches are bf16 or fp16")
        if not _on_gpu(t):
            raise ValueError(f"{name} must be on the GPU")
    if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype or k_cache.device != v_cache.device:
        raise ValueError("k_cache and v_cache must share shape, dtype and device")
    D = k_cache.shape[3]
    assert _is_pow2(D), f"Head dim D={D} must be a power of two"
    if D not in HEAD_DIMS:
        raise ValueError(f"head dim {D}: the cache operators take {HEAD_DIMS}")
    for t, name in zip((k_cache, v_cache), names):
        _check_cache_layout(t, name)
    return k_cache.shape


def _check_writable(k_cache, v_cache):
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if any(t.shape[d] > 1 and t.stride(d) == 0 for d in range(3)):
            raise ValueError(f"{name} is updated in place: it must not be an expanded tensor")
    if k_cache.data_ptr() == v_cache.data_ptr():
        raise ValueError("k_cache and v_cache are updated in place: they must not share memory")


def _check_queries(q, k_cache):
    """q as [B, Hq, T, D] and whether it came as [B, Hq, D]."""
    squeeze = q.dim() == 3
    q4 = q.unsqueeze(2) if squeeze else q
    if q4.dim() != 4:
        raise ValueError("q must be [B, Hq, T, D] or [B, Hq, D]")
    B, Hkv, _, D = k_cache.shape
    if q4.shape[0] != B or q4.shape[3] != D or q4.shape[2] < 1:
        raise ValueError(f"q {tuple(q.shape)} does not match the cache {tuple(k_cache.shape)}")
    Hq = q4.shape[1]
    assert Hq % Hkv == 0, f"Hq={Hq} must be divisible by Hkv={Hkv}"
    if q.dtype != k_cache.dtype:
        raise ValueError("q and the caches must share one dtype")
    if q.device != k_cache.device:
        raise ValueError("q and the caches must be on the same GPU device")
    return _kernel_layout(q4), squeeze


def _lens(cache_seqlens, B, device):
    lens = torch.as_tensor(cache_seqlens, device=device)
    if lens.shape != (B,):
        raise ValueError(f"cache_seqlens must have shape ({B},)")
    if lens.is_floating_point():
        raise ValueError("cache_seqlens must hold integers")
    return lens.to(torch.int32).contiguous()


def _check_weights(weights, B, Hkv, cap, device):
    if not torch.is_tensor(weights) or tuple(weights.shape) != (B, Hkv, cap):
        raise ValueError(f"weights must be [B, Hkv, capacity] = {(B, Hkv, cap)}")
    if weights.dtype != torch.float32 or weights.device != device or (cap > 1 and weights.stride(2) != 1):
        raise ValueError("weights must be fp32 on the caches' device with a contiguous last dimension")


def _int32(t, shape, device, name):
    t = torch.as_tensor(t, device=device)
    if tuple(t.shape) != tuple(shape) or t.is_floating_point():
        raise ValueError(f"{name} must hold integers of shape {tuple(shape)}")
    return t.to(torch.int32).contiguous()


def _launch(entry: str, args, device):
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        _lib.check(getattr(_lib.lib(), entry)(ctypes.byref(args), ctypes.c_void_p(stream)), entry)


def tree_mask_from_parents(parents) -> torch.Tensor:
    """The mask of a drafted tree: ``parents[i]`` is node i's parent (a node
    before it) or negative for a node that follows the cached prefix itself.
    ``mask[i, j]`` is true where j is i or an ancestor of i.  ``parents`` is
    ``[T]`` or ``[B, T]``, a host tensor or nested list; the result is a bool
    tensor on the host."""
    par = torch.as_tensor(parents)
    if par.dim() not in (1, 2) or par.is_floating_point() or par.shape[-1] < 1:
        raise ValueError("parents must hold integers of shape [T] or [B, T]")
    if par.is_cuda:
        raise ValueError("parents must be on the host")
    T = par.shape[-1]
    if bool((par >= torch.arange(T)).any()):
        raise ValueError("a node's parent must come before it")
    rows = par.reshape(-1, T)
    mask = torch.zeros(rows.shape[0], T, T, dtype=torch.bool)
    batch = torch.arange(rows.shape[0])
    for i in range(T):
        up = rows[:, i]
        mask[:, i] = mask[batch, up.clamp_min(0)] & (up >= 0)[:, None]
        mask[:, i, i] = True
    return mask if par.dim() == 2 else mask[0]


def ssa_tree_num_splits(B: int, Hq: int, Hkv: int, capacity: int, nodes: int, num_splits: int = 0) -> int:
    """Key splits ``ssa_tree_attention`` uses (``num_splits`` = 0: its own choice)."""
    return int(_lib.lib().ssa_tree_num_splits(B, Hq, Hkv, capacity, nodes, num_splits))


def check_tree_call(q, k_cache, v_cache, tree_mask):
    """Raises for the queries, caches and mask that ``ssa_tree_attention`` does not
    take; (q as [B, Hq, T, D], whether it came as [B, Hq, D], the mask on q's device)."""
    B = _check_caches(k_cache, v_cache)[0]
    q4, squeeze = _check_queries(q, k_cache)
    T = q4.shape[2]
    if T > MAX_TREE_NODES:
        raise ValueError(f"a tree has at most {MAX_TREE_NODES} tokens, got {T}")
    mask = torch.as_tensor(tree_mask, device=q.device)
    if tuple(mask.shape) not in ((T, T), (B, T, T)):
        raise ValueError(f"tree_mask must be [{T}, {T}] or [{B}, {T}, {T}], got {tuple(mask.shape)}")
    return q4, squeeze, mask


def ssa_tree_attention(q, k_cache, v_cache, cache_seqlens, tree_mask, softmax_scale, ssa_n, ssa_b, num_splits=0,
                       return_m=False):
    """The tokens of a drafted tree attend the cache, in one pass over it.

    ``q`` is ``[B, Hq, T, D]`` (``[B, Hq, D]`` for one token), T up to 1024; the
    keys and values of the T drafted tokens are already the last T rows that
    ``cache_seqlens`` counts, token j of sequence b at row
    ``cache_seqlens[b] - T + j``.  Token i attends every row before the tree's
    and token j's where ``tree_mask[i, j]`` (bool ``[T, T]``, or ``[B, T, T]``
    for a tree of its own per sequence; ``tree_mask_from_parents`` makes one; in
    another type, what is not 0 is seen, so an additive mask is none).  A
    lower triangular mask gives the causal attention of T consecutive tokens.
    Returns ``out`` shaped like ``q`` (and ``m [B, Hq, T]`` fp32 with
    ``return_m``).  A token that sees nothing gets ``out = 0``, ``m = -inf``; a
    sequence shorter than T holds the tree's last tokens only.  What a token does
    not see does not reach it, NaN and infinities included.  A sequence's results
    do not depend on the others', and are bitwise reproducible for one set of
    sizes and ``num_splits``.
    """
    if q.is_cuda:
        r = _lib.native().tree(q, k_cache, v_cache, cache_seqlens, tree_mask, softmax_scale, ssa_n, ssa_b, num_splits,
                               bool(return_m), *_current())
        if r is not None:
            r = _native_result(r, "ssa_tree_attention")
            return r if return_m else r[0]
    q4, squeeze, mask = check_tree_call(q, k_cache, v_cache, tree_mask)
    B, Hq, T, D = q4.shape
    Hkv, cap = k_cache.shape[1:3]
    mask = (mask if mask.dtype in (torch.bool, torch.uint8) else mask != 0).contiguous()
    lens = _lens(cache_seqlens, B, q.device)
    n32, b32 = _scalar(ssa_n, q.device), _scalar(ssa_b, q.device)
    out = torch.empty((B, Hq, T, D), dtype=q.dtype, device=q.device)
    m = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device) if return_m else None
    ws_bytes = int(_lib.lib().ssa_tree_workspace_bytes(B, Hq, Hkv, cap, D, T, int(num_splits)))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes > 0 else None
    args = _lib.TreeArgs(
        _t4(q4), _t4(k_cache), _t4(v_cache), _t4(out),
        m.data_ptr() if m is not None else None, lens.data_ptr(), mask.data_ptr(), T * T if mask.dim() == 3 else 0,
        n32.data_ptr(), b32.data_ptr(), B, Hq, Hkv, cap, D, _DTYPES[q.dtype], T, int(num_splits),
        float(softmax_scale), ws.data_ptr() if ws is not None else None,
    )
    _launch("ssa_tree_attention", args, q.device)
    if squeeze:
        out, m = out.squeeze(2), (m.squeeze(2) if m is not None else None)
    return (out, m) if return_m else out


def ssa_key_weights(q, k_cache, m, cache_seqlens, weights, softmax_scale, ssa_n, ssa_b):
    """Adds to every cached key's weight the attention that the last queries paid to it.

    ``q`` is ``[B, Hq, T, D]`` (``[B, Hq, D]`` for one), query t of sequence b at
    position ``cache_seqlens[b] - T + t`` and seeing the rows up to its own;
    ``m`` ``[B, Hq, T]`` (or ``[B, Hq]``) holds the normalisers that the
    attention returned for these queries (``ssa_flash_attn_forward``,
    ``ssa_decode_attention`` or ``ssa_tree_attention`` with ``return_m``).
    ``weights`` fp32 ``[B, Hkv, capacity]`` is updated in place and returned:
    row j of head h gains the sum of the probabilities that the queries of h's
    group gave it.  A query whose m is -inf adds nothing.
    """
    if q.is_cuda:
        r = _lib.native().key_weights(q, k_cache, m, cache_seqlens, weights, softmax_scale, ssa_n, ssa_b, *_current())
        if r is not None:
            _native_result(r, "ssa_key_weights")
            return weights
    B, Hkv, cap, D = _check_caches(k_cache, k_cache)
    q4, squeeze = _check_queries(q, k_cache)
    Hq, T = q4.shape[1], q4.shape[2]
    if T > cap:
        raise ValueError(f"{T} queries cannot stand in a cache of {cap} rows")
    if not torch.is_tensor(m) or tuple(m.shape) not in ((B, Hq, T),) + (((B, Hq),) if T == 1 else ()):
        raise ValueError(f"m must be [B, Hq, T] = {(B, Hq, T)}")
    if m.device != q.device:
        raise ValueError("m must be on the caches' device")
    m32 = m.to(torch.float32).contiguous()
    _check_weights(weights, B, Hkv, cap, q.device)
    lens = _lens(cache_seqlens, B, q.device)
    n32, b32 = _scalar(ssa_n, q.device), _scalar(ssa_b, q.device)
    ws_bytes = int(_lib.lib().ssa_key_weights_workspace_bytes(B, Hq, Hkv, cap, T))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes > 0 else None
    args = _lib.KeyWeightsArgs(
        _t4(q4), _t4(k_cache), m32.data_ptr(), weights.data_ptr(), weights.stride(0), weights.stride(1),
        lens.data_ptr(), n32.data_ptr(), b32.data_ptr(), B, Hq, Hkv, cap, D, _DTYPES[q.dtype], T,
        float(softmax_scale), ws.data_ptr() if ws is not None else None,
    )
    _launch("ssa_key_weights", args, q.device)
    return weights


def ssa_cache_evict(k_cache, v_cache, cache_seqlens, weights, keep, sinks=0, recent=0):
    """Cuts every cache that holds more than ``keep`` rows to ``keep`` of them.

    Kept are the first ``sinks`` and the last ``recent`` rows (together at most
    ``keep``) and, of the others, those of largest ``weights`` (fp32
    ``[B, Hkv, capacity]``; of equal weights the lower row, NaN lowest); each
    (sequence, kv-head) keeps rows of its own, in their order.  The rows move in
    place; ``cache_seqlens`` and ``weights`` are left as they are, and the new
    ones are returned: ``(lens int32 [B], weights [B, Hkv, capacity], kept int32
    [B, Hkv, keep])``, the weights of the rows that stayed followed by zeros and
    the rows they came from followed by -1.
    """
    if k_cache.is_cuda:
        r = _lib.native().evict(k_cache, v_cache, cache_seqlens, weights, keep, sinks, recent, *_current())
        if r is not None:
            return _native_result(r, "ssa_cache_evict")
    B, Hkv, cap, D = _check_caches(k_cache, v_cache)
    _check_writable(k_cache, v_cache)
    dev = k_cache.device
    _check_weights(weights, B, Hkv, cap, dev)
    keep, sinks, recent = int(keep), int(sinks), int(recent)
    if not 1 <= keep <= cap or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"keep must be 1 .. {cap} and hold sinks + recent, got keep={keep} sinks={sinks} "
                         f"recent={recent}")
    lens = _lens(cache_seqlens, B, dev)
    new = torch.empty(B, dtype=torch.int32, device=dev)
    w_out = torch.empty((B, Hkv, cap), dtype=torch.float32, device=dev)
    kept = torch.empty((B, Hkv, keep), dtype=torch.int32, device=dev)
    args = _lib.CacheEvictArgs(
        _t4(k_cache), _t4(v_cache), weights.data_ptr(), weights.stride(0), weights.stride(1), lens.data_ptr(),
        new.data_ptr(), w_out.data_ptr(), kept.data_ptr(), B, Hkv, cap, D, _DTYPES[k_cache.dtype], keep, sinks, recent,
    )
    _launch("ssa_cache_evict", args, dev)
    return new, w_out, kept


def ssa_cache_accept(k_cache, v_cache, cache_seqlens, path, accepted, nodes):
    """Accepts a path of a drafted tree of ``nodes`` tokens, the cache's last rows.

    With first = ``cache_seqlens[b] - nodes``, row ``first + path[b, i]`` moves
    to row ``first + i`` for i below ``accepted[b]``; the new lengths,
    first + accepted, are returned (int32 ``[B]``; ``cache_seqlens`` is left as it
    is).  ``path`` is int32 ``[B, depth]`` with depth at most ``nodes``, in any
    order; entries at and behind ``accepted[b]`` are not used.  On the device
    ``accepted`` is clamped to 0 .. depth and path entries to 0 .. nodes - 1; a
    sequence shorter than ``nodes`` is left as it is.
    """
    if k_cache.is_cuda:
        r = _lib.native().accept(k_cache, v_cache, cache_seqlens, path, accepted, nodes, *_current())
        if r is not None:
            return _native_result(r, "ssa_cache_accept")[0]
    B, Hkv, cap, D = _check_caches(k_cache, v_cache)
    _check_writable(k_cache, v_cache)
    dev, nodes = k_cache.device, int(nodes)
    path = torch.as_tensor(path, device=dev)
    depth = path.shape[1] if path.dim() == 2 else 0
    if not 1 <= nodes <= MAX_TREE_NODES or not 1 <= depth <= nodes:
        raise ValueError(f"path must be [B, depth] with 1 <= depth <= nodes <= {MAX_TREE_NODES}, got "
                         f"{tuple(path.shape)} and nodes={nodes}")
    path = _int32(path, (B, depth), dev, "path")
    accepted = _int32(accepted, (B,), dev, "accepted")
    lens = _lens(cache_seqlens, B, dev)
    new = torch.empty(B, dtype=torch.int32, device=dev)
    args = _lib.CacheAcceptArgs(
        _t4(k_cache), _t4(v_cache), lens.data_ptr(), path.data_ptr(), accepted.data_ptr(), new.data_ptr(),
        B, Hkv, cap, D, _DTYPES[k_cache.dtype], nodes, depth,
    )
    _launch("ssa_cache_accept", args, dev)
    return new
