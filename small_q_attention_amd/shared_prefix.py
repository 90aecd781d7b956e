"""Small-q attention for batches whose sequences begin with the same pages: answers sampled
from one prompt, requests under one system prompt or over one document. The shared pages are
read once for each group of sequences and not once for each sequence.

That takes a few microseconds more than attention over the whole rows of few and short
sequences, and pays from about 32K tokens saved on, (sequences - 1) * shared tokens: the same
result comes from ``cuda.paged_mtp_attention`` or a window over everything.

:func:`plan_shared_prefix` says which sequences share how many pages, once for as long as
that stays; :func:`paged_attention_shared_prefix` is the attention call, with the result of
attention over the whole block tables. It runs on the current stream of the query's device,
allocates nothing but its result and a workspace, never synchronises and can be captured in a
HIP graph (keep the plan as long as the graph). A plan serves any stream, and may be dropped
while its eager calls still wait to run.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from . import scaled_cache as sc
from .cuda import HEAD_DIMS, SUPPORTED_PAGE_SIZES, _tracing
from .masks import as_words
from .windowed import check_apart, check_call, check_factors, take_workspace, whole_pages


class SharedPrefixPlan:
    """What :func:`plan_shared_prefix` returns: ``shape`` (batch, q_len, query heads, kv
    heads, head_dim, page_size), ``groups`` as given, and their table on ``device``."""

    def __init__(self, shape, groups, device, table):
        self.shape, self.groups, self.device, self.table = shape, groups, device, table
        # What traced calls pass on, and the most table columns that a group shares.
        self.flat = [x for g in groups for x in g]
        self.most_pages = max([pages for _, count, pages in groups if count > 1] + [0])
        self.known = sc.Layouts()
        self.streams = set()  # of the eager calls so far


def plan_shared_prefix(groups, batch: int, q_len: int, num_query_heads: int, num_kv_heads: int,
                       head_dim: int, page_size: int, device=None) -> SharedPrefixPlan:
    """Plan for a batch and the prefixes its sequences share.

    ``groups``: ``(first, count, pages)`` triples, in ascending order and apart: sequences
    ``first .. first + count - 1`` begin with the same ``pages`` entries of their block
    tables. Sequences of no group share nothing. The plan holds for as long as the groups and
    what they share stay, whatever the sequences' lengths and the pages' ids; calls with
    another shape refuse it. One small copy to ``device`` (``None``: the current one).
    """
    groups = [tuple(int(x) for x in g) for g in groups]
    shape = tuple(int(x) for x in (batch, q_len, num_query_heads, num_kv_heads, head_dim,
                                   page_size))
    b, q, hq, hkv, d, page = shape
    if min(b, q, hq, hkv) <= 0 or hq % hkv:
        raise ValueError("batch, q_len and heads must be positive, query heads a multiple of kv "
                         "heads")
    if d not in HEAD_DIMS:
        raise ValueError("this build supports head_dim 64, 128 or 256")
    if page not in SUPPORTED_PAGE_SIZES:
        raise ValueError("this build supports page_size 16, 32, 64, 128 or 256")
    most = 32 if d == 256 else 64
    if q * (hq // hkv) > most:
        raise ValueError(f"Q * (Hq / Hkv) must be at most {most} at head_dim {d}")
    end = 0
    for g in groups:
        if len(g) != 3 or g[0] < end or g[1] <= 0 or g[2] < 0 or g[0] + g[1] > b:
            raise ValueError("groups are (first, count, pages), in ascending order, apart and "
                             f"within the batch; got {g}")
        if g[2] * page >= 2**30:
            raise ValueError("block-table rows must be under 2^30 tokens")
        end = g[0] + g[1]
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError("the plan's device must be a GPU")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    groups = tuple(groups)
    most = max([pages for *_, pages in groups] + [1])
    _, _, table = _lib.plan_shared_prefix(device.index, groups, shape, 0, 0, most)
    table = torch.tensor(table, dtype=torch.int32).to(device)
    return SharedPrefixPlan(shape, groups, device, table)


def _check(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens, words,
           plan, out, workspace_buffer):
    check_call(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens, words,
               out, workspace_buffer)
    shape = (*query.shape[:3], key_cache.shape[2], query.shape[3], key_cache.shape[1])
    if shape != plan.shape:
        raise ValueError(f"the plan was made for (batch, q_len, query heads, kv heads, head_dim, "
                         f"page_size) {plan.shape}, the call has {tuple(shape)}")
    if plan.device != query.device:
        raise ValueError(f"the plan lives on {plan.device}, query on {query.device}")
    if plan.most_pages > block_tables.shape[1]:
        raise ValueError(f"the plan shares {plan.most_pages} pages, block_tables rows hold "
                         f"{block_tables.shape[1]}")


def _plan_call(query, key_cache, key_scale, block_tables, words, groups, max_seq_len):
    b, q_len, hq, d = query.shape
    plan, need, _ = _lib.plan_shared_prefix(
        query.device.index, groups, (b, q_len, hq, key_cache.shape[2], d, key_cache.shape[1]),
        _lib.dtype_code(key_cache.dtype), max_seq_len, block_tables.shape[1])
    return plan, need, _lib.part_fields(query, key_cache, key_scale, block_tables, words)


def hold_table(table, stream, device, streams=None):
    """Keep a plan's table for the calls on ``stream``, the current one: dropped with the plan
    before they have run, its memory goes to nobody until they have. Once for each of
    ``streams``. (Not under graph capture: there the caller keeps the plan.)"""
    if streams is not None and stream in streams:
        return
    _, capturing = _lib._CUDA_STATE or _lib._cuda_state(torch)
    if capturing():
        return
    table.record_stream(torch.cuda.current_stream(device))
    if streams is not None:
        streams.add(stream)


def run_shared_prefix(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens,
                      words, groups, table, scale, out_scale, max_seq_len, out, workspace,
                      known=None, streams=None):
    """Plan and launch a checked call (``groups``, ``table``, ``streams``: a plan's; ``known``:
    the call's :func:`_plan_call`)."""
    plan, need, fields = known or _plan_call(query, key_cache, key_scale, block_tables, words,
                                             groups, max_seq_len)
    stream = _lib.raw_stream(query.device.index)
    hold_table(table, stream, query.device, streams)
    workspace = take_workspace(workspace, need, query, stream)
    if out is None:
        out = torch.empty_like(query)
    _lib.launch_shared_prefix(query, out, key_cache, value_cache, key_scale, value_scale,
                              block_tables, seq_lens, words, plan, table, scale, out_scale,
                              workspace, stream, fields)
    return out


def paged_attention_shared_prefix(query, key_cache, value_cache, block_tables, seq_lens,
                                  plan: SharedPrefixPlan, key_scale=None, value_scale=None,
                                  max_seq_len: int = 0, scale: Optional[float] = None,
                                  out_scale: float = 1.0, mask=None, out=None,
                                  workspace_buffer=None):
    """Small-q attention of a batch whose sequences share prefixes.

    ``query`` ``[B, Q, Hq, D]`` (fp16 or bf16), caches ``[P, page, Hkv, D]`` of the query's
    type, of ``torch.float8_e4m3fn``, or codes with ``key_scale``/``value_scale``;
    ``block_tables`` ``[B, max_pages]`` and ``seq_lens`` ``[B]`` int32 as for the other
    attention calls: whole tables and whole lengths, shared pages and draft tokens counted.
    Row ``i`` of a sequence sees the tokens before its draft block and, of the block, those
    up to its own or those ``mask`` names (the packed draft mask of
    :mod:`small_q_attention_amd.masks`); rows that see no token are 0. A group's shared pages
    are taken from the table row of its first sequence that is long enough for all of its
    rows to lie behind them; the entries of the others' rows are not read there. A sequence
    that is not (a padded batch's) goes over its own row from the start.

    ``max_seq_len`` > 0 only sizes the call (0: the block table's width), and with it the
    last bits of a result may change; a call of another layout or number of 16-token pages is
    planned anew, 50 to 300 us on the host, so a loop better passes a bound that stays for many
    calls. ``scale`` is the softmax scale (``None``: ``D **
    -0.5``), ``out_scale`` multiplies the output. Over bf16 caches the
    probabilities of shared pages are rounded once to bf16 (2^-8 of each; a row's weights still
    add up to one) for groups of more than 64 rows of a kv head (32 at head_dim 256), and kept to
    2^-16 otherwise.
    ``workspace_buffer``: a caller's buffer for the partial rows; ``None`` takes one kept per
    host thread and stream, or, under graph capture, one of the graph's own. A graph reads
    the plan's table: the plan is kept for as long as the graph is replayed. Returns ``out``
    (``[B, Q, Hq, D]``).
    """
    if query.dim() != 4:
        raise ValueError("query must be a contiguous [B, Q, Hq, D] tensor")
    if not isinstance(plan, SharedPrefixPlan):
        raise ValueError("plan must come from plan_shared_prefix()")
    scale, out_scale = check_factors(scale, out_scale, query.shape[3])
    words = None if mask is None else as_words(mask, query.shape[0], query.shape[1])
    max_seq_len = whole_pages(max_seq_len)
    if _tracing():
        _check(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens, words,
               plan, out, workspace_buffer)
        from . import _op  # noqa: F401  (registers the ops)

        res = torch.ops.sqa.paged_attention_shared_prefix(
            query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens, words,
            plan.flat, plan.table, scale, out_scale, max_seq_len)
        return res if out is None else out.copy_(res)
    layout = sc.layout
    seen = (layout(query), layout(key_cache), layout(value_cache), layout(key_scale),
            layout(value_scale), layout(block_tables), layout(seq_lens), layout(words),
            layout(out), workspace_buffer is None or workspace_buffer.device, max_seq_len)
    known = plan.known.get(seen)
    if known is None:
        _check(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens, words,
               plan, out, workspace_buffer)
        known = plan.known.keep(seen, sc.on_device(query.device, _plan_call, query, key_cache,
                                                   key_scale, block_tables, words, plan.groups,
                                                   max_seq_len))
    sc.check_aligned(16, query, key_cache, value_cache)
    check_apart(query, out)
    return sc.on_device(query.device, run_shared_prefix, query, key_cache, value_cache, key_scale,
                        value_scale, block_tables, seq_lens, words, plan.groups, plan.table, scale,
                        out_scale, max_seq_len, out, workspace_buffer, known, plan.streams)


__all__ = ["SharedPrefixPlan", "plan_shared_prefix", "paged_attention_shared_prefix"]
