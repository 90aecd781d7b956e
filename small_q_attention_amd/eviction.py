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
from .masks import as_words

_HALF = (torch.float16, torch.bfloat16)


def _check_weights(weights, batch, hkv, what="weights"):
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[0] != batch \
            or weights.shape[1] != hkv or weights.shape[2] == 0 or weights.stride(2) != 1:
        raise ValueError(f"{what} must be float32 [{batch}, {hkv}, tokens] with a contiguous last "
                         "dimension")
    sc.check_distinct(weights, what)


def _check_scaled(cache, *scales):
    for s in scales:
        if s is not None and cache.dtype not in sc.CODE_DTYPES:
            raise ValueError("scales belong to caches of torch.float8_e4m3fn or torch.int8")
        if s is None and cache.dtype is torch.int8:
            raise ValueError("int8 caches need scales")
        if s is not None:
            sc.check_scale(s, cache, "a cache's scale")


_WEIGHS, _EVICTIONS = sc.Layouts(), sc.Layouts()


def run_weights(query, key_cache, key_scale, block_tables, seq_lens, words, weights, scale,
                max_seq_len, known=None):
    """Plan and launch a checked call (``known``: its :func:`_weights_plan`)."""
    need, fields = known or _weights_plan(query, key_cache, key_scale, block_tables, words,
                                          weights, max_seq_len)
    index = query.device.index
    stream = _lib.raw_stream(index)
    workspace = _lib.workspace_for(need, query, index, stream)
    _lib.launch_weights(query, key_cache, key_scale, block_tables, seq_lens, words, weights, scale,
                        max_seq_len, workspace, stream, fields)


def _weights_plan(query, key_cache, key_scale, block_tables, words, weights, max_seq_len):
    batch, q_len, hq, d = query.shape
    need = _lib.weights_workspace_bytes(query.device.index, batch, q_len, hq, key_cache.shape[2], d,
                                        max_seq_len,
                                        block_tables.shape[1] * (key_cache.shape[1] // 16),
                                        _lib.dtype_code(key_cache.dtype))
    return need, _lib.weights_fields(query, key_cache, key_scale, block_tables, words, weights,
                                     max_seq_len)


def _check_accumulate(query, key_cache, block_tables, seq_lens, weights, key_scale, words):
    sc.check_pool(key_cache)
    sc.check_query(query, key_cache)
    if key_cache.dtype != query.dtype and key_cache.dtype not in sc.CODE_DTYPES:
        raise ValueError("key_cache must hold the query's type, torch.float8_e4m3fn or torch.int8")
    _check_scaled(key_cache, key_scale)
    batch = query.shape[0]
    sc.check_batch(batch, block_tables, seq_lens)
    _check_weights(weights, batch, key_cache.shape[2])
    sc.check_on(query.device, key_cache=key_cache, key_scale=key_scale, block_tables=block_tables,
                seq_lens=seq_lens, weights=weights, mask=words, query=query)


def accumulate_attention_weights(query, key_cache, block_tables, seq_lens, weights, key_scale=None,
                                 max_seq_len: int = 0, scale: Optional[float] = None, mask=None):
    """Add up the attention weights of one call, in place.

    ``query`` ``[B, Q, Hq, D]``, ``mask`` and the visible tokens as in
    :func:`scaled_cache.paged_attention_scaled`. ``weights`` ``[B, Hkv, T]`` float32:
    ``weights[b, h, t]`` grows by the softmax probabilities that the ``Q * Hq / Hkv`` rows
    of kv head ``h`` give token ``t``. The last ``Q`` tokens' weights are set, not added to:
    they start with this call, whatever a draft that was taken back left there. Tokens from
    ``T`` on are not recorded, entries past a sequence's end not touched. ``max_seq_len``
    > 0 promises that no sequence is longer and sizes the workspace, as the block table's
    width does without it (scores of up to 1 GiB where that is wide). Returns ``weights``.
    """
    if query.dim() != 4:
        raise ValueError("query must be a contiguous [B, Q, Hq, D] tensor")
    scale = sc.check_softmax_scale(scale, query.shape[3])
    words = None if mask is None else as_words(mask, query.shape[0], query.shape[1])
    max_seq_len = min(max(int(max_seq_len), 0), 2**31 - 1)
    if _tracing():
        _check_accumulate(query, key_cache, block_tables, seq_lens, weights, key_scale, words)
        from . import _op  # noqa: F401  (registers the ops)

        torch.ops.sqa.accumulate_attention_weights(query, key_cache, key_scale, block_tables,
                                                   seq_lens, words, weights, scale, max_seq_len)
        return weights
    layout = sc.layout
    seen = (layout(query), layout(key_cache), layout(key_scale), layout(block_tables),
            layout(seq_lens), layout(weights), layout(words), max_seq_len)
    known = _WEIGHS.get(seen)
    if known is None:
        _check_accumulate(query, key_cache, block_tables, seq_lens, weights, key_scale, words)
        known = _WEIGHS.keep(seen, sc.on_device(query.device, _weights_plan, query, key_cache,
                                                key_scale, block_tables, words, weights,
                                                max_seq_len))
    sc.check_aligned(16, query, key_cache)
    sc.on_device(query.device, run_weights, query, key_cache, key_scale, block_tables, seq_lens,
                 words, weights, scale, max_seq_len, known)
    return weights


def launch_evict(weights, new_weights, kept, seq_lens, new_lens, source, into, block_tables,
                 new_tables, budget, sink, recent, fields=None):
    """Launch a checked call on the current stream."""
    _lib.launch_evict(weights, new_weights, kept, seq_lens, new_lens, source, into, block_tables,
                      new_tables, budget, sink, recent, _lib.raw_stream(weights.device.index),
                      fields)


def _check_evict(weights, source, block_tables, seq_lens, new_block_tables, budget, sink, recent,
                 into, new_weights):
    key_cache, value_cache, key_scale, value_scale = source
    sc.check_pool(key_cache)
    if key_cache.dtype not in _HALF + sc.CODE_DTYPES:
        raise ValueError("caches must hold float16, bfloat16, float8_e4m3fn or int8")
    sc.check_same_layout(key_cache, value_cache, "key_cache and value_cache")
    if (key_scale is None) != (value_scale is None):
        raise ValueError("key_scale and value_scale come together")
    if len(into) != 4 or into[0] is None or into[1] is None:
        raise ValueError("into must be (key_cache, value_cache[, key_scale, value_scale])")
    sc.check_pool(into[0], "into's key_cache")
    sc.check_same_layout(into[0], into[1], "into's caches")
    sc.check_distinct(into[0], "into's caches")
    if into[0].dtype != key_cache.dtype or into[0].shape[1:] != key_cache.shape[1:]:
        raise ValueError("into's caches must match in type, page size, kv heads and head_dim")
    if (into[2] is None) != (key_scale is None) or (into[3] is None) != (key_scale is None):
        raise ValueError("into needs scales where the cache has them, and only there")
    _check_scaled(key_cache, key_scale, value_scale)
    _check_scaled(into[0], into[2], into[3])
    if key_scale is not None:
        sc.check_same_layout(key_scale, value_scale, "key_scale and value_scale")
        sc.check_same_layout(into[2], into[3], "into's scales")
        sc.check_distinct(into[2], "into's scales")
    for cache in (key_cache, into[0]):
        if any(x * cache.element_size() % 16 for x in cache.stride()[:3]):
            raise ValueError("cache strides must be multiples of 16 bytes")
    batch, hkv = seq_lens.shape[0] if seq_lens.dim() == 1 else 0, key_cache.shape[2]
    if batch == 0:
        raise ValueError("seq_lens must be a [batch] tensor and not empty")
    sc.check_batch(batch, block_tables, seq_lens)
    sc.check_batch(batch, new_block_tables, seq_lens, "new_block_tables")
    _check_weights(weights, batch, hkv)
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
    call uses, each of them once (the old ones may be shared by several), or to the caches of
    ``into``:
    ``(key_cache, value_cache)`` of the same type, page size and heads, with
    ``(..., key_scale, value_scale)`` for scaled ones. In scaled caches a new block takes the
    largest scale among the blocks its tokens come from, and codes of other blocks are
    rounded again. Tokens from ``T`` on weigh 0 (the last ``recent`` stay all the same); lengths
    past the table's width are held to it.

    ``weights`` may be written in place: ``new_weights=weights`` (a buffer that overlaps it in
    another way may not be given); ``None`` returns new ones, ``[B, Hkv, budget]``: no wider
    than what is kept, so a loop that goes on to add up the weights of later tokens gives a
    buffer with room for them.

    Returns ``(new_lens [B] int32, new_weights, kept [B, Hkv, budget] int32)``: the lengths
    ``min(seq_lens, budget)``, the moved weights (0 past them) and the positions the tokens
    had before (-1 past them).
    """
    budget, sink, recent = int(budget), int(sink), int(recent)
    source = (key_cache, value_cache, key_scale, value_scale)
    if into is None:
        into = source
    elif len(into) == 2:
        into = (*into, None, None)
    if _tracing():
        _check_evict(weights, source, block_tables, seq_lens, new_block_tables, budget, sink,
                     recent, into, new_weights)
        from . import _op  # noqa: F401  (registers the ops)

        kept, new_lens, new_weights = _results(weights, seq_lens, budget, new_weights)
        torch.ops.sqa.evict_by_weight(weights, *source, block_tables, seq_lens, new_block_tables,
                                      *into, new_weights, new_lens, kept, budget, sink, recent)
        return new_lens, new_weights, kept
    layout = sc.layout
    seen = (layout(weights), layout(new_weights), layout(key_cache), layout(value_cache),
            layout(key_scale), layout(value_scale), layout(block_tables), layout(seq_lens),
            layout(new_block_tables), *[layout(t) for t in into], budget, sink, recent)
    fields = _EVICTIONS.get(seen)
    if fields is None:
        _check_evict(weights, source, block_tables, seq_lens, new_block_tables, budget, sink,
                     recent, into, new_weights)
    sc.check_aligned(16, key_cache, value_cache, into[0], into[1])
    sc.check_apart(*into)
    kept, new_lens, new_weights = _results(weights, seq_lens, budget, new_weights)
    if fields is None:
        fields = _EVICTIONS.keep(seen, _lib.evict_fields(
            weights, new_weights, source, into, block_tables, new_block_tables, budget, sink,
            recent))
    sc.on_device(weights.device, launch_evict, weights, new_weights, kept, seq_lens, new_lens,
                 source, into, block_tables, new_block_tables, budget, sink, recent, fields)
    return new_lens, new_weights, kept


def _results(weights, seq_lens, budget, new_weights):
    shape, device = (weights.shape[0], weights.shape[1], budget), weights.device
    kept = torch.empty(shape, dtype=torch.int32, device=device)
    if new_weights is None:
        new_weights = torch.empty(shape, dtype=torch.float32, device=device)
    return kept, torch.empty_like(seq_lens), new_weights


__all__ = ["accumulate_attention_weights", "evict_by_weight"]
