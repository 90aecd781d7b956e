"""Small-q attention over a window: every row sees the last tokens up to its own and the
first few of its sequence (attention sinks), so a stream of any length costs what its
window costs.

:func:`paged_attention_windowed` takes caches of the query's type, of
``torch.float8_e4m3fn`` (per-tensor scales go into ``scale`` and ``out_scale``) and, with
``key_scale``/``value_scale``, codes with block scales
(:mod:`small_q_attention_amd.scaled_cache`). It runs on the current stream of the query's
device, allocates nothing but its result and a workspace, never synchronises and can be
captured in a HIP graph.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from . import scaled_cache as sc
from .cuda import _tracing
from .masks import as_words

_KNOWN = sc.Layouts()


def check_caches(query, key_cache, value_cache, key_scale, value_scale):
    """The caches of a call: of the query's type, e4m3, or codes with scales."""
    sc.check_pool(key_cache)
    sc.check_same_layout(key_cache, value_cache, "key_cache and value_cache")
    if (key_scale is None) != (value_scale is None):
        raise ValueError("key_scale and value_scale come together")
    if key_scale is not None:
        if key_cache.dtype not in sc.CODE_DTYPES:
            raise ValueError("scales belong to caches of torch.float8_e4m3fn or torch.int8")
        sc.check_scale(key_scale, key_cache)
        sc.check_scale(value_scale, key_cache, "value_scale")
        sc.check_same_layout(key_scale, value_scale, "key_scale and value_scale")
    elif key_cache.dtype is torch.int8:
        raise ValueError("caches of torch.int8 need key_scale and value_scale")
    elif key_cache.dtype not in (query.dtype, torch.float8_e4m3fn):
        raise ValueError("caches must hold the query's type or torch.float8_e4m3fn (or, with "
                         "scales, torch.int8)")


def check_call(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens, words,
               out, workspace_buffer):
    sc.check_query(query, key_cache)
    check_caches(query, key_cache, value_cache, key_scale, value_scale)
    sc.check_batch(query.shape[0], block_tables, seq_lens)
    sc.check_on(query.device, key_cache=key_cache, value_cache=value_cache, key_scale=key_scale,
                value_scale=value_scale, block_tables=block_tables, seq_lens=seq_lens, mask=words,
                out=out, workspace_buffer=workspace_buffer, query=query)
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype
                            or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor shaped and typed like query")


_LARGEST = 2.0 ** 128 - 2.0 ** 103  # numbers from here on are no float32


def check_factors(scale, out_scale, d):
    """The softmax scale (``None``: ``d ** -0.5``) and the output's factor, as floats that 32
    bits hold."""
    scale, out_scale = sc.check_softmax_scale(scale, d), float(out_scale)
    if not 2.0 ** -150 < scale < _LARGEST or not abs(out_scale) < _LARGEST:
        raise ValueError("scale must be positive and finite and out_scale finite, in 32 bits")
    return scale, out_scale


def whole_pages(max_seq_len) -> int:
    """``max_seq_len`` as the plans look at it, in whole pages of 16 tokens: a loop whose longest
    sequence grows by one plans again every sixteenth call."""
    return min((max(int(max_seq_len), 0) + 15) // 16 * 16, 2**31 - 16)


def check_apart(query, out):
    """ValueError for a result that takes some of the queries' place: they are read until the
    end. (Both are contiguous, of one size.)"""
    if out is not None and abs(out.data_ptr() - query.data_ptr()) < query.nbytes:
        raise ValueError("out must not be query, nor overlap it")


def take_workspace(workspace_buffer, need, query, stream):
    """The caller's buffer, checked, or one kept for the stream (``None`` where none is
    needed)."""
    if workspace_buffer is None:
        return _lib.workspace_for(need, query, query.device.index, stream) if need else None
    if workspace_buffer.numel() * workspace_buffer.element_size() < need \
            or not workspace_buffer.is_contiguous():
        raise ValueError(f"workspace_buffer must be contiguous and hold at least {need} bytes "
                         "for this batch")
    return workspace_buffer


def _plan(query, key_cache, key_scale, block_tables, words, window, sink, max_seq_len):
    b, q_len, hq, d = query.shape
    page, hkv = key_cache.shape[1], key_cache.shape[2]
    cut = _lib.plan_windowed(query.device.index, b, q_len, hq, hkv, d, window, sink, max_seq_len,
                             block_tables.shape[1] * (page // 16),
                             _lib.dtype_code(key_cache.dtype))
    return (cut, _lib.workspace_bytes(b, q_len, hq, hkv, d, cut[0], cut[1]),
            _lib.part_fields(query, key_cache, key_scale, block_tables, words))


def run_windowed(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens,
                 words, window, sink, scale, out_scale, max_seq_len, out, workspace, known=None):
    """Plan and launch a checked call (``known``: its :func:`_plan`)."""
    cut, need, fields = known or _plan(query, key_cache, key_scale, block_tables, words, window,
                                       sink, max_seq_len)
    stream = _lib.raw_stream(query.device.index)
    workspace = take_workspace(workspace, need, query, stream)
    if out is None:
        out = torch.empty_like(query)
    _lib.launch_windowed(query, out, key_cache, value_cache, key_scale, value_scale, block_tables,
                         seq_lens, words, window, sink, scale, out_scale, cut, workspace, stream,
                         fields)
    return out


def paged_attention_windowed(query, key_cache, value_cache, block_tables, seq_lens, window: int,
                             sink: int = 0, key_scale=None, value_scale=None, max_seq_len: int = 0,
                             scale: Optional[float] = None, out_scale: float = 1.0, mask=None,
                             out=None, workspace_buffer=None):
    """Small-q attention over the last ``window`` tokens and the first ``sink``.

    ``query`` ``[B, Q, Hq, D]`` (fp16 or bf16; ``Q * Hq / Hkv <= 64``, 32 at head_dim 256),
    caches ``[P, page, Hkv, D]`` (or views of an interleaved one), ``block_tables`` ``[B,
    max_pages]`` and ``seq_lens`` ``[B]`` int32. Draft row ``i`` of sequence ``b`` stands at
    ``p = seq_lens[b] - Q + i``; of the tokens that it sees without a window (those before
    the draft block, and of the block those up to its own or those ``mask`` names, the packed
    draft mask of :mod:`small_q_attention_amd.masks`) it sees token ``t`` if ``t < sink`` or
    ``t > p - window``: its own counts as one of the ``window``. Positions are slots of the
    sequence, also under a draft tree. Rows that see no token are 0. Pages that no row sees
    are not read, and their table entries may hold anything (a page that has left the window
    can be given back); an id outside the pool among the others stands for page 0. A value
    that is not finite reaches the rows that see its token and no others.

    ``key_scale``/``value_scale`` ``[P, Hkv]`` float32: block scales of e4m3 or int8 codes,
    within the ranges of :func:`scaled_cache.paged_attention_scaled`. ``max_seq_len`` > 0
    only sizes the call (0: the block table's width), and with it the last bits of a result
    may change; a call of another layout, window or number of 16-token pages is planned anew,
    about 10 us on the host. ``scale`` is the softmax scale (``None``: ``D ** -0.5``), ``out_scale``
    multiplies the output. ``workspace_buffer``: a caller's buffer for the split partials;
    ``None`` takes one kept per host thread and stream, or, under graph capture, one of the
    graph's own. Returns ``out`` (``[B, Q, Hq, D]``).
    """
    if query.dim() != 4:
        raise ValueError("query must be a contiguous [B, Q, Hq, D] tensor")
    scale, out_scale = check_factors(scale, out_scale, query.shape[3])
    window, sink = int(window), int(sink)
    if window <= 0 or sink < 0:
        raise ValueError("window must be positive and sink not negative")
    window, sink = min(window, 2**31 - 1), min(sink, 2**31 - 1)
    words = None if mask is None else as_words(mask, query.shape[0], query.shape[1])
    max_seq_len = whole_pages(max_seq_len)
    if _tracing():
        check_call(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens,
                   words, out, workspace_buffer)
        from . import _op  # noqa: F401  (registers the ops)

        res = torch.ops.sqa.paged_attention_windowed(
            query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens, words,
            window, sink, scale, out_scale, max_seq_len)
        return res if out is None else out.copy_(res)
    layout = sc.layout
    seen = (layout(query), layout(key_cache), layout(value_cache), layout(key_scale),
            layout(value_scale), layout(block_tables), layout(seq_lens), layout(words),
            layout(out), workspace_buffer is None or workspace_buffer.device, window, sink,
            max_seq_len)
    known = _KNOWN.get(seen)
    if known is None:
        check_call(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens,
                   words, out, workspace_buffer)
        known = _KNOWN.keep(seen, sc.on_device(query.device, _plan, query, key_cache, key_scale,
                                               block_tables, words, window, sink, max_seq_len))
    sc.check_aligned(16, query, key_cache, value_cache)
    check_apart(query, out)
    return sc.on_device(query.device, run_windowed, query, key_cache, value_cache, key_scale,
                        value_scale, block_tables, seq_lens, words, window, sink, scale,
                        out_scale, max_seq_len, out, workspace_buffer, known)


__all__ = ["paged_attention_windowed"]
