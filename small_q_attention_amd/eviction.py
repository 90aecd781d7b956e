"""Thinning out a paged cache by the attention its tokens receive.

* :func:`accumulate_attention_weights` adds up, for every cached token and kv head, the
  softmax probabilities a call's query rows give it;
* :func:`evict_by_weight` keeps the first and the last tokens of every sequence and the
  heaviest of the others, and moves them together on new pages.

Both take caches of the query's 16-bit type, e4m3, and e4m3 or int8 with block scales
(:mod:`small_q_attention_amd.scaled_cache`), as ``[P, page, Hkv, D]`` pools or views. They
run on the current stream of the tensors' device, without a host synchronisation, and can
be captured in a HIP graph.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from . import scaled_cache as sc
from .cuda import _tracing

_HALF = (torch.float16, torch.bfloat16)


def _check_weights(weights, batch, hkv, what="weights"):
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[0] != batch \
            or weights.shape[1] != hkv or weights.shape[2] == 0 or weights.stride(2) != 1:
        raise ValueError(f"{what} must be float32 [{batch}, {hkv}, tokens] with a contiguous last "
                         "dimension")


def _check_scaled(cache, *scales):
    for s in scales:
        if s is not None and cache.dtype not in sc.CODE_DTYPES:
            raise ValueError("scales belong to caches of torch.float8_e4m3fn or torch.int8")
        if s is None and cache.dtype is torch.int8:
            raise ValueError("int8 caches need scales")
        if s is not None:
            sc.check_scale(s, cache, "a cache's scale")


def run_weights(query, key_cache, key_scale, block_tables, seq_lens, words, weights, scale,
                max_seq_len):
    """Plan and launch a checked call."""
    batch, q_len, hq, d = query.shape
    index = query.device.index
    need = _lib.weights_workspace_bytes(index, batch, q_len, hq, key_cache.shape[2], d, max_seq_len,
                                        block_tables.shape[1] * (key_cache.shape[1] // 16),
                                        _lib.dtype_code(key_cache.dtype))
    stream = _lib.raw_stream(index)
    workspace = _lib.workspace_for(need, query, index, stream)
    _lib.launch_weights(query, key_cache, key_scale, block_tables, seq_lens, words, weights, scale,
                        max_seq_len, workspace, stream)


def accumulate_attention_weights(query, key_cache, block_tables, seq_lens, weights, key_scale=None,
                                 max_seq_len: int = 0, scale: Optional[float] = None, mask=None):
    """Add up the attention weights of one call, in place.

    ``query`` ``[B, Q, Hq, D]``, ``mask`` and the visible tokens as in
    :func:`scaled_cache.paged_attention_scaled`. ``weights`` ``[B, Hkv, T]`` float32:
    ``weights[b, h, t]`` grows by the softmax probabilities that the ``Q * Hq / Hkv`` rows
    of kv head ``h`` give token ``t``. The last ``Q`` tokens' weights are set, not added to:
    they start with this call, whatever a draft that was taken back left there. Tokens from
    ``T`` on are not recorded, entries past a sequence's end not touched. ``max_seq_len``
    > 0 promises that no sequence is longer. Returns ``weights``.
    """
    sc.check_pool(key_cache)
    sc.check_query(query, key_cache)
    if key_cache.dtype != query.dtype and key_cache.dtype not in sc.CODE_DTYPES:
        raise ValueError("key_cache must hold the query's type, torch.float8_e4m3fn or torch.int8")
    _check_scaled(key_cache, key_scale)
    batch, q_len = query.shape[:2]
    sc.check_batch(batch, block_tables, seq_lens)
    _check_weights(weights, batch, key_cache.shape[2])
    device = query.device
    sc.check_on(device, key_cache=key_cache, key_scale=key_scale, block_tables=block_tables,
                seq_lens=seq_lens, weights=weights)
    scale = sc.check_softmax_scale(scale, query.shape[3])
    words = sc.mask_words(mask, batch, q_len, device)
    max_seq_len = max(int(max_seq_len), 0)
    if _tracing():
        from . import _op  # noqa: F401  (registers the ops)

        torch.ops.sqa.accumulate_attention_weights(query, key_cache, key_scale, block_tables,
                                                   seq_lens, words, weights, scale, max_seq_len)
        return weights
    sc.on_device(device, lambda: run_weights(query, key_cache, key_scale, block_tables, seq_lens,
                                             words, weights, scale, max_seq_len))
    return weights


def run_evict(weights, new_weights, source, block_tables, seq_lens, into, new_tables, budget, sink,
              recent):
    """Allocate what a checked call returns and launch it."""
    kept = torch.empty(weights.shape[0], weights.shape[1], budget, dtype=torch.int32,
                       device=weights.device)
    new_lens = torch.empty_like(seq_lens)
    if new_weights is None:
        new_weights = torch.empty(kept.shape, dtype=torch.float32, device=weights.device)
    _lib.launch_evict(weights, new_weights, kept, seq_lens, new_lens, source, into, block_tables,
                      new_tables, budget, sink, recent, _lib.raw_stream(weights.device.index))
    return new_lens, new_weights, kept


def evict_by_weight(weights, key_cache, value_cache, block_tables, seq_lens, new_block_tables,
                    budget: int, sink: int = 0, recent: int = 0, key_scale=None, value_scale=None,
                    into=None, new_weights=None):
    """Keep at most ``budget`` tokens of every sequence, for each kv head its own.

    Kept are the first ``sink`` tokens, the last ``recent``, and the heaviest of those
    between by ``weights`` ``[B, Hkv, T]`` (NaN counts as the lightest; of equal ones the
    earlier stays). They move, in their order, to positions 0, 1, ... on the pages of
    ``new_block_tables`` ``[B, W]`` (``W`` pages must hold ``budget`` tokens); a sequence
    within the budget moves whole. Keys keep whatever position they were rotated to.

    The new pages belong to the same pool, and then must be pages that no sequence of the
    call uses (the old ones may be shared by several), or to the caches of ``into``:
    ``(key_cache, value_cache)`` of the same type, page size and heads, with
    ``(..., key_scale, value_scale)`` for scaled ones. In scaled caches a new block takes the
    largest scale among the blocks its tokens come from, and codes of other blocks are
    rounded again. ``weights`` may be written in place: ``new_weights=weights``; ``None``
    returns new ones, ``[B, Hkv, budget]``. ``T`` and the table bound the lengths that are
    looked at.

    Returns ``(new_lens [B] int32, new_weights, kept [B, Hkv, budget] int32)``: the lengths
    ``min(seq_lens, budget)``, the moved weights (0 past them) and the positions the tokens
    had before (-1 past them).
    """
    sc.check_pool(key_cache)
    if key_cache.dtype not in _HALF + sc.CODE_DTYPES:
        raise ValueError("caches must hold float16, bfloat16, float8_e4m3fn or int8")
    sc.check_same_layout(key_cache, value_cache, "key_cache and value_cache")
    if (key_scale is None) != (value_scale is None):
        raise ValueError("key_scale and value_scale come together")
    source = (key_cache, value_cache, key_scale, value_scale)
    into = source if into is None else tuple(into) + (None,) * (4 - len(tuple(into)))
    if len(into) != 4 or into[0] is None or into[1] is None:
        raise ValueError("into must be (key_cache, value_cache[, key_scale, value_scale])")
    sc.check_pool(into[0], "into's key_cache")
    sc.check_same_layout(into[0], into[1], "into's caches")
    if into[0].dtype != key_cache.dtype or into[0].shape[1:] != key_cache.shape[1:]:
        raise ValueError("into's caches must match in type, page size, kv heads and head_dim")
    if (into[2] is None) != (key_scale is None) or (into[3] is None) != (key_scale is None):
        raise ValueError("into needs scales where the cache has them, and only there")
    _check_scaled(key_cache, key_scale, value_scale)
    _check_scaled(into[0], into[2], into[3])
    if key_scale is not None:
        sc.check_same_layout(key_scale, value_scale, "key_scale and value_scale")
        sc.check_same_layout(into[2], into[3], "into's scales")
    for cache in (key_cache, into[0]):
        if any(x * cache.element_size() % 16 for x in cache.stride()[:3]):
            raise ValueError("cache strides must be multiples of 16 bytes")
    if sc.misaligned(value_cache, 16) or sc.misaligned(into[1], 16):
        raise ValueError("caches must be 16-byte aligned")
    batch, hkv = seq_lens.shape[0] if seq_lens.dim() == 1 else 0, key_cache.shape[2]
    if batch == 0:
        raise ValueError("seq_lens must be a [batch] tensor and not empty")
    sc.check_batch(batch, block_tables, seq_lens)
    sc.check_batch(batch, new_block_tables, seq_lens, "new_block_tables")
    _check_weights(weights, batch, hkv)
    budget, sink, recent = int(budget), int(sink), int(recent)
    if budget <= 0 or sink < 0 or recent < 0 or sink + recent > budget:
        raise ValueError("budget must be positive and hold sink + recent tokens")
    if budget > new_block_tables.shape[1] * key_cache.shape[1]:
        raise ValueError("new_block_tables must have pages for budget tokens")
    if new_weights is not None:
        _check_weights(new_weights, batch, hkv, "new_weights")
        if new_weights.shape[2] < budget:
            raise ValueError("new_weights must hold budget tokens")
    sc.check_on(weights.device, new_weights=new_weights, key_cache=key_cache,
                value_cache=value_cache, key_scale=key_scale, value_scale=value_scale,
                block_tables=block_tables, seq_lens=seq_lens, new_block_tables=new_block_tables,
                into_key_cache=into[0], into_value_cache=into[1], into_key_scale=into[2],
                into_value_scale=into[3])
    if _tracing():
        raise ValueError("evict_by_weight is not traced: call it outside torch.compile")
    return sc.on_device(weights.device, lambda: run_evict(
        weights, new_weights, source, block_tables, seq_lens, into, new_block_tables, budget, sink,
        recent))


__all__ = ["accumulate_attention_weights", "evict_by_weight"]
