"""SSA self-attention module on the MI355X kernels, without Megatron.

Mirrors ``SSATritonAttention`` (training/train/train_ssa_triton/SSA/ssa_triton_attention.py):

* constructor arguments and parameter names (``ssa_n_raw``, ``ssa_b_raw`` or the
  ``ssa_b`` buffer, ``ssa_n`` buffer when not learnable; :99-113), so reference
  checkpoints load unchanged;
* softmax scale 1/sqrt(head_dim), divided by the layer number under query-key
  layer scaling (:91-97);
* forward(query, key, value [S, B, H, D]) -> context [S, B, Hq * D] (:132-202),
  dropout applied to the attention output, never inside the op (:115-130).

Differences, both at the boundary: the [S, B, H, D] inputs are handed to the
kernels as permuted views (no copies; the reference forces contiguous copies
in production, ``force_contiguous_qkv``), and the kernel writes its output in
[S, B, H, D] memory order, so the final [S, B, Hq * D] reshape is a view;
packed sequences (``packed_seq_params`` with ``cu_seqlens_q`` and
``max_seqlen_q``, tensors [T, H, D] or [T, 1, H, D]) run on the varlen path,
which the reference rejects (:154-156).

Generation: ``SSAKVCache`` + ``SSAAttention.forward_decode`` run one token
per step against the cached keys and values (the decode kernel), where the
reference's generation loop re-runs the whole prefix through the forward for
every token (training/train/train_ssa_triton/generate_triton.py:315-331); the
result is the same causal attention row.  A drafted tree of tokens is checked
in one step (``forward_tree``, then ``SSAKVCache.accept`` for the path that was
right), and a cache that tracks its keys' accumulated attention weights
(``track_weights``) can be cut to a budget (``SSAKVCache.evict``).
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import nn

from .ssa_cache_ops import (HEAD_DIMS, check_tree_call, ssa_cache_accept, ssa_cache_evict, ssa_key_weights,
                            ssa_tree_attention)
from .ssa_flash_attention import ssa_flash_attention, ssa_flash_attention_varlen
from .ssa_hip_kernel import ssa_decode_attention, ssa_flash_attn_forward


class SSAKVCache:
    """Keys and values of one attention layer for generation.

    ``k`` / ``v`` are ``[B, Hkv, capacity, D]`` (the decode kernel's layout);
    ``seqlens`` (int32 ``[B]``, on the device) counts the cached tokens of each
    sequence.  Appends write at each sequence's own length without a host
    synchronisation; positions past ``capacity`` are clamped to its last row,
    so the caller sizes the cache for the longest generation.

    With ``track_weights``, ``weights`` (fp32 ``[B, Hkv, capacity]``) holds the
    attention that the queries so far paid to every cached key (0 behind the
    sequence); ``SSAAttention`` keeps it up to date, and ``evict`` cuts the
    cache by it (bf16 and fp16, head dims 32, 64 and 128).
    """

    def __init__(self, batch: int, heads_kv: int, capacity: int, head_dim: int, dtype=torch.bfloat16,
                 device="cuda", track_weights: bool = False):
        if track_weights and (dtype not in (torch.bfloat16, torch.float16) or head_dim not in HEAD_DIMS):
            raise ValueError(f"weights are tracked in caches of bf16 or fp16 with head dims {HEAD_DIMS}, not of "
                             f"{dtype} with {head_dim}")
        self.k = torch.zeros(batch, heads_kv, capacity, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.seqlens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.capacity = capacity
        self.weights = (torch.zeros(batch, heads_kv, capacity, dtype=torch.float32, device=device)
                        if track_weights else None)
        self._drafted = None  # (q, m, scale, n, b) of the last drafted tree, for the weights of its accepted path

    @torch.no_grad()
    def append(self, key: torch.Tensor, value: torch.Tensor) -> None:
        """Append ``T`` new tokens per sequence: key / value ``[B, Hkv, T, D]``.
        The cache holds their values: no gradient reaches them through it."""
        self._drafted = None
        B, _, T, _ = key.shape
        pos = self.seqlens.long().unsqueeze(1) + torch.arange(T, device=key.device).unsqueeze(0)
        pos = pos.clamp_(max=self.capacity - 1)
        bidx = torch.arange(B, device=key.device).unsqueeze(1).expand(B, T)
        # advanced indices on dims 0 and 2 -> the indexed view is [B, T, Hkv, D]
        self.k[bidx, :, pos] = key.transpose(1, 2).to(self.k.dtype)
        self.v[bidx, :, pos] = value.transpose(1, 2).to(self.v.dtype)
        self.seqlens += T

    def add_weights(self, q: torch.Tensor, m: torch.Tensor, softmax_scale, ssa_n, ssa_b) -> None:
        """Adds the attention that the last queries (``[B, Hq, T, D]`` or ``[B, Hq,
        D]``, ``m`` their normalisers) paid to the cached keys
        (``ssa_key_weights``)."""
        if self.weights is None:
            raise ValueError("the cache does not track weights (track_weights=True)")
        ssa_key_weights(q, self.k, m, self.seqlens, self.weights, softmax_scale, ssa_n, ssa_b)

    def evict(self, keep: int, sinks: int = 0, recent: int = 0) -> torch.Tensor:
        """Cuts every sequence of more than ``keep`` rows to ``keep`` of them, by
        weight, the first ``sinks`` and last ``recent`` rows in any case
        (``ssa_cache_evict``); returns the rows that stayed, int32 ``[B, Hkv,
        keep]``, -1 behind the last."""
        if self.weights is None:
            raise ValueError("the cache does not track weights (track_weights=True)")
        self._drafted = None
        lens, weights, kept = ssa_cache_evict(self.k, self.v, self.seqlens, self.weights, keep, sinks, recent)
        self.seqlens.copy_(lens)
        self.weights.copy_(weights)
        return kept

    def accept(self, path: torch.Tensor, accepted: torch.Tensor, nodes: int) -> None:
        """Keeps of the last ``nodes`` rows, a drafted tree's, the first
        ``accepted[b]`` nodes of ``path[b]``, in that order
        (``ssa_cache_accept``).  A tracking cache gains the attention that the
        accepted tokens paid."""
        drafted = self._drafted
        if drafted is not None and drafted[0].shape[2] != nodes:
            raise ValueError(f"the last tree had {drafted[0].shape[2]} nodes, not {nodes}")
        path = torch.as_tensor(path, device=self.k.device)
        accepted = torch.as_tensor(accepted, device=self.k.device)
        weighs = self.weights is not None and drafted is not None
        held = self.seqlens.clamp(max=self.capacity) >= nodes if weighs else None
        self.seqlens.copy_(ssa_cache_accept(self.k, self.v, self.seqlens, path, accepted, nodes))
        self._drafted = None
        if not weighs:
            return
        q, m, scale, n, b = drafted
        # the path's queries at the end of the sequence, rows that were not accepted before them
        depth = path.shape[1]
        count = accepted.long().clamp(0, depth).masked_fill(~held, 0)
        step = torch.arange(depth, device=path.device)[None, :] - (depth - count)[:, None]
        node = path.long().clamp(0, nodes - 1).gather(1, step.clamp_min(0))
        at = node[:, None, :].expand(-1, q.shape[1], -1)
        rows = q.gather(2, at[..., None].expand(-1, -1, -1, q.shape[3]))
        norm = m.gather(2, at).masked_fill((step < 0)[:, None, :], -math.inf)
        ssa_key_weights(rows, self.k, norm, self.seqlens, self.weights, scale, n, b)


class SSAAttention(nn.Module):
    def __init__(
        self,
        num_attention_heads: int,
        num_query_groups: Optional[int] = None,
        kv_channels: int = 128,
        layer_number: int = 1,
        softmax_scale: Optional[float] = None,
        apply_query_key_layer_scaling: bool = False,
        attention_dropout: float = 0.0,
        ssa_n: float = 1.5,
        ssa_b: float = 0.8,
        learnable_ssa: bool = True,
        learnable_b: bool = False,
        causal: bool = True,
    ):
        super().__init__()
        self.num_heads = num_attention_heads
        self.num_query_groups = num_query_groups or num_attention_heads
        if self.num_heads % self.num_query_groups != 0:
            raise ValueError("num_attention_heads must be a multiple of num_query_groups")
        self.head_dim = kv_channels
        self.hidden_size = kv_channels * num_attention_heads
        self.layer_number = max(1, layer_number)
        self.causal = causal
        self.learnable_ssa = learnable_ssa
        self.learnable_b = learnable_b
        self.softmax_scale = 1.0 / math.sqrt(kv_channels) if softmax_scale is None else softmax_scale
        if apply_query_key_layer_scaling:
            self.softmax_scale /= self.layer_number
        if learnable_ssa:
            self.ssa_n_raw = nn.Parameter(torch.tensor(float(ssa_n)))
            if learnable_b:
                self.ssa_b_raw = nn.Parameter(torch.tensor(float(ssa_b)))
            else:
                self.register_buffer("ssa_b", torch.tensor(float(ssa_b)))
        else:
            self.register_buffer("ssa_n", torch.tensor(float(ssa_n)))
            self.register_buffer("ssa_b", torch.tensor(float(ssa_b)))
        self.dropout_p = attention_dropout
        self.attention_dropout = nn.Dropout(attention_dropout)

    def get_ssa_params(self):
        if self.learnable_ssa:
            return self.ssa_n_raw, (self.ssa_b_raw if self.learnable_b else self.ssa_b)
        return self.ssa_n, self.ssa_b

    def forward(self, query, key, value, attention_mask=None, packed_seq_params=None):
        """query [S, B, Hq, D], key/value [S, B, Hkv, D] -> context [S, B, Hq * D].

        With ``packed_seq_params`` (``cu_seqlens_q``, ``max_seqlen_q``): tensors
        [T, H, D] or [T, 1, H, D] -> context [T, Hq * D] (or [T, 1, Hq * D]).
        ``attention_mask`` is ignored (the causal mask is applied in the kernel).
        """
        n, b = self.get_ssa_params()
        if packed_seq_params is not None:
            squeeze = query.dim() == 4
            q, k, v = (t.squeeze(1) if squeeze else t for t in (query, key, value))
            ctx = ssa_flash_attention_varlen(q, k, v, packed_seq_params.cu_seqlens_q,
                                             packed_seq_params.max_seqlen_q, self.softmax_scale, n, b, self.causal)
            if self.training and self.dropout_p > 0:
                ctx = self.attention_dropout(ctx)
            ctx = ctx.reshape(ctx.shape[0], -1)
            return ctx.unsqueeze(1) if squeeze else ctx
        S, B = query.shape[0], query.shape[1]
        # [S, B, H, D] -> [B, H, S, D] views: the kernels read the strides in place
        q, k, v = (t.permute(1, 2, 0, 3) for t in (query, key, value))
        ctx = ssa_flash_attention(q, k, v, self.softmax_scale, n, b, self.causal, self.dropout_p, self.training)
        if self.training and self.dropout_p > 0:
            ctx = self.attention_dropout(ctx)
        # the output has the strides of q, i.e. [S, B, H, D] memory order: views only
        return ctx.permute(2, 0, 1, 3).reshape(S, B, -1)

    def forward_decode(self, query, key, value, cache: SSAKVCache):
        """One generation step.  query [1, B, Hq, D], key/value [1, B, Hkv, D]
        (the new token) -> context [1, B, Hq * D]; the key and value are
        appended to ``cache`` first, so the token attends itself and the
        cached prefix (causal)."""
        if query.shape[0] != 1:
            raise ValueError("forward_decode takes one new token per sequence ([1, B, H, D])")
        n, b = self.get_ssa_params()
        cache.append(key.permute(1, 2, 0, 3), value.permute(1, 2, 0, 3))
        track = cache.weights is not None
        ctx = ssa_decode_attention(query[0], cache.k, cache.v, cache.seqlens, self.softmax_scale, n, b,
                                   return_m=track)
        if track:
            ctx, m = ctx
            cache.add_weights(query[0], m, self.softmax_scale, n, b)
        return ctx.reshape(1, query.shape[1], -1)

    @torch.no_grad()
    def forward_prompt(self, query, key, value, cache: SSAKVCache, window: Optional[int] = None):
        """A prompt into an empty cache of at least its length: query [S, B, Hq, D],
        key/value [S, B, Hkv, D] -> context [S, B, Hq * D] of the dense causal forward, without
        gradients; keys and values go to ``cache``, and a tracking cache gains
        the attention that the last ``window`` tokens (None: all) paid."""
        n, b = self.get_ssa_params()
        if query.shape[0] > cache.capacity:
            raise ValueError(f"a prompt of {query.shape[0]} tokens in a cache of {cache.capacity} rows")
        w = query.shape[0] if window is None else min(window, query.shape[0])
        weighs = cache.weights is not None and w > 0
        if weighs and query.dtype != cache.k.dtype:
            raise ValueError(f"queries of {query.dtype} for the weights of a cache of {cache.k.dtype}")
        q, k, v = (t.permute(1, 2, 0, 3) for t in (query, key, value))
        out, m = ssa_flash_attn_forward(q, k, v, self.softmax_scale, n, b, True)
        cache.append(k, v)
        if weighs:
            cache.add_weights(q[:, :, -w:], m[:, :, -w:], self.softmax_scale, n, b)
        return out.permute(2, 0, 1, 3).reshape(query.shape[0], query.shape[1], -1)

    @torch.no_grad()
    def forward_tree(self, query, key, value, cache: SSAKVCache, tree_mask):
        """One step over a drafted tree of T tokens per sequence, without gradients.
        query [T, B, Hq, D], key/value [T, B, Hkv, D] -> context [T, B, Hq * D]; keys
        and values are appended to ``cache``, and token i attends the cached prefix and the
        tokens that ``tree_mask`` ([T, T] or [B, T, T]) gives it.  Then
        ``cache.accept`` keeps the path that was right.  A call that is refused
        leaves the cache as it was."""
        n, b = self.get_ssa_params()
        if query.shape[0] > cache.capacity:
            raise ValueError(f"a tree of {query.shape[0]} tokens in a cache of {cache.capacity} rows")
        tree_mask = torch.as_tensor(tree_mask, device=query.device)
        check_tree_call(query.permute(1, 2, 0, 3), cache.k, cache.v, tree_mask)  # before anything is appended
        cache.append(key.permute(1, 2, 0, 3), value.permute(1, 2, 0, 3))
        q = query.detach().permute(1, 2, 0, 3)  # kept for accept, without the graph behind it
        track = cache.weights is not None
        ctx = ssa_tree_attention(q, cache.k, cache.v, cache.seqlens, tree_mask, self.softmax_scale, n, b,
                                 return_m=track)
        if track:
            ctx, m = ctx
            cache._drafted = (q, m, self.softmax_scale, n, b)
        return ctx.permute(2, 0, 1, 3).reshape(query.shape[0], query.shape[1], -1)
