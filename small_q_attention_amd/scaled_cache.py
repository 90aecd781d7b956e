"""KV caches held in 8 bits with a scale for each page and kv head.

``key_cache``/``value_cache`` are ``[P, page, Hkv, D]`` pools (or views of one, as the
halves of an interleaved NHD or HND cache) of ``torch.float8_e4m3fn`` or ``torch.int8``;
``key_scale``/``value_scale`` are ``[P, Hkv]`` float32. Code ``c`` of page ``p`` and head
``h`` stands for ``c * scale[p, h]``.

* :func:`append_scaled_kv` quantises new tokens into the cache;
* :func:`paged_attention_scaled` is small-q attention over it.

The scale of a block is the largest magnitude of its tokens over 448 (e4m3) or 127
(int8). Scales must be finite and not negative (0: a block of zeros); the calls do not
look at them. Both calls run on the current stream of the tensors' device, allocate
nothing but what they return and a workspace, and can be captured in a HIP graph.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .cuda import HEAD_DIMS, SUPPORTED_PAGE_SIZES, _tracing
from .masks import as_words

CODE_DTYPES = (torch.float8_e4m3fn, torch.int8)


def check_aligned(n, *tensors):
    """ValueError unless the tensors start on ``n``-byte boundaries (not for traced ones,
    which have no address: the library checks it when the graph runs)."""
    for t in tensors:
        if t.data_ptr() % n:
            raise ValueError(f"a tensor of {tuple(t.shape)} does not start on a {n}-byte boundary")


def check_on(device, **tensors):
    """ValueError unless every tensor lives on the GPU ``device``: raw pointers of host or
    other-device memory must never reach a kernel."""
    if device.type != "cuda":
        raise ValueError("the tensors must be GPU tensors")
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be a GPU tensor on {device}")


def check_pool(cache, what="key_cache"):
    """A ``[P, page, Hkv, D]`` view the kernels can read by its strides."""
    if cache.dim() != 4 or cache.shape[0] == 0 or cache.shape[2] == 0:
        raise ValueError(f"{what} must be [P, page, Hkv, D] and not empty")
    if cache.shape[1] not in SUPPORTED_PAGE_SIZES:
        raise ValueError("this build supports page_size 16, 32, 64, 128 or 256")
    if cache.shape[3] not in HEAD_DIMS:
        raise ValueError("this build supports head_dim 64, 128 or 256")
    s = cache.stride()
    if s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8:
        raise ValueError(f"{what} needs a contiguous head dimension and other strides in "
                         "multiples of 8 elements")


def check_same_layout(a, b, what):
    if b.shape != a.shape or b.dtype != a.dtype or b.stride() != a.stride():
        raise ValueError(f"{what} must match in shape, type and strides")


def check_distinct(t, what):
    """ValueError for a tensor that is written and has elements in one place (expanded)."""
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{what} must not be an expanded tensor: it is written")


def check_apart(key_cache, value_cache, key_scale, value_scale):
    """ValueError for one cache, or one tensor of scales, given for keys and values both: they
    are written."""
    if key_cache.data_ptr() == value_cache.data_ptr() or (
            key_scale is not None and key_scale.data_ptr() == value_scale.data_ptr()):
        raise ValueError("keys and values each need a cache and scales of their own: they are "
                         "written")


def check_scale(scale, cache, what="key_scale"):
    if scale.dtype != torch.float32 or tuple(scale.shape) != (cache.shape[0], cache.shape[2]):
        raise ValueError(f"{what} must be float32 [{cache.shape[0]}, {cache.shape[2]}]")


def check_batch(batch, block_tables, seq_lens, name="block_tables"):
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise ValueError(f"{name} and seq_lens must be int32")
    if block_tables.dim() != 2 or block_tables.shape[0] != batch or block_tables.shape[1] == 0 \
            or not block_tables.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{batch}, max_pages] tensor")
    if seq_lens.dim() != 1 or seq_lens.shape[0] != batch or not seq_lens.is_contiguous():
        raise ValueError(f"seq_lens must be a contiguous [{batch}] tensor")


def check_query(query, cache):
    if query.dim() != 4 or not query.is_contiguous() or query.shape[0] == 0 \
            or query.shape[1] == 0:
        raise ValueError("query must be a contiguous [B, Q, Hq, D] tensor")
    if query.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("query must be float16 or bfloat16")
    hq, d, hkv = query.shape[2], query.shape[3], cache.shape[2]
    if d != cache.shape[3] or hq == 0 or hq % hkv:
        raise ValueError("query needs the cache's head_dim and a multiple of its kv heads")
    most = 32 if d == 256 else 64
    if query.shape[1] * (hq // hkv) > most:
        raise ValueError(f"Q * (Hq / Hkv) must be at most {most} at head_dim {d}")


def check_softmax_scale(scale, d):
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale must be positive and finite")
    return scale


def on_device(device, call, *args):
    """``call(*args)`` with ``device`` as the current one."""
    current, _ = _lib._CUDA_STATE or _lib._cuda_state(torch)
    if device.index == current():
        return call(*args)
    with torch.cuda.device(device):
        return call(*args)


class Layouts(dict):
    """What the checks of an entry point found for the layouts (shapes, strides, types and
    devices, nothing of the data) of a call's tensors: a serving loop makes the same kind
    of call again and again, and the checks cost more than the launch. Bounded."""

    def keep(self, key, value):
        if len(self) >= 1024:
            self.clear()
        self[key] = value
        return value


def layout(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _check_cache(key_cache, value_cache, key_scale, value_scale):
    check_pool(key_cache)
    if key_cache.dtype not in CODE_DTYPES:
        raise ValueError("caches must hold torch.float8_e4m3fn or torch.int8")
    check_same_layout(key_cache, value_cache, "key_cache and value_cache")
    check_scale(key_scale, key_cache)
    check_scale(value_scale, key_cache, "value_scale")
    check_same_layout(key_scale, value_scale, "key_scale and value_scale")


def append_scaled_kv(key, value, key_cache, value_cache, key_scale, value_scale, block_tables,
                     seq_lens, new_lens: Optional[torch.Tensor] = None) -> None:
    """Quantise new tokens into the cache, in place.

    ``key``/``value`` ``[B, Q, Hkv, D]`` (fp16 or bf16, any strides in multiples of 8
    elements with a contiguous head dimension). Sequence ``b`` gets its first
    ``new_lens[b]`` tokens (``None``: all ``Q``) at positions ``seq_lens[b] - new_lens[b]``
    on: ``seq_lens`` counts them already, as it does the draft tokens in the attention
    calls. A block's scale is the largest magnitude among its new tokens over 448 (e4m3)
    or 127 (int8), and at least its old scale where earlier tokens of the sequence stay in
    the page; where it grows, their codes are rounded again. Slots past the sequence's end
    and pages outside the pool or the table are left as they are. Infinities count as the
    type's largest finite value; a NaN does not count and is stored as NaN (e4m3) or 0
    (int8). No page may be written twice in one call, by two sequences or by two entries of
    one table row.
    """
    if _tracing():
        _check_append(key, value, key_cache, value_cache, key_scale, value_scale, block_tables,
                      seq_lens, new_lens)
        from . import _op  # noqa: F401  (registers the ops)

        torch.ops.sqa.append_scaled_kv(key, value, key_cache, value_cache, key_scale, value_scale,
                                       block_tables, seq_lens, new_lens)
        return
    seen = (layout(key), layout(value), layout(key_cache), layout(value_cache), layout(key_scale),
            layout(value_scale), layout(block_tables), layout(seq_lens), layout(new_lens))
    fields = _APPENDS.get(seen)
    if fields is None:
        _check_append(key, value, key_cache, value_cache, key_scale, value_scale, block_tables,
                      seq_lens, new_lens)
        fields = _APPENDS.keep(seen, _lib.append_fields(key, value, key_cache, key_scale,
                                                        block_tables))
    check_aligned(16, key, value, key_cache, value_cache)
    check_apart(key_cache, value_cache, key_scale, value_scale)
    on_device(key.device, _launch_append, key, value, key_cache, value_cache, key_scale,
              value_scale, block_tables, seq_lens, new_lens, fields)


_APPENDS, _ATTENTIONS = Layouts(), Layouts()


def _launch_append(key, value, key_cache, value_cache, key_scale, value_scale, block_tables,
                   seq_lens, new_lens, fields):
    _lib.launch_append(key, value, key_cache, value_cache, key_scale, value_scale, block_tables,
                       seq_lens, new_lens, _lib.raw_stream(key.device.index), fields)


def _check_append(key, value, key_cache, value_cache, key_scale, value_scale, block_tables,
                  seq_lens, new_lens):
    if key.dim() != 4 or value.shape != key.shape or key.shape[0] == 0 or key.shape[1] == 0:
        raise ValueError("key and value must be [B, Q, Hkv, D] tensors of one shape")
    if key.dtype not in (torch.float16, torch.bfloat16) or value.dtype != key.dtype:
        raise ValueError("key and value must both be float16 or bfloat16")
    _check_cache(key_cache, value_cache, key_scale, value_scale)
    check_distinct(key_cache, "key_cache")
    check_distinct(key_scale, "key_scale")
    if tuple(key.shape[2:]) != tuple(key_cache.shape[2:]):
        raise ValueError("key and value need the cache's kv heads and head_dim")
    for t in (key, value):
        s = t.stride()
        if s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8:
            raise ValueError("key and value need a contiguous head dimension and other strides "
                             "in multiples of 8 elements")
    batch = key.shape[0]
    check_batch(batch, block_tables, seq_lens)
    if new_lens is not None and (new_lens.dtype != torch.int32 or new_lens.shape != seq_lens.shape
                                 or not new_lens.is_contiguous()):
        raise ValueError(f"new_lens must be a contiguous int32 [{batch}] tensor")
    check_on(key.device, value=value, key_cache=key_cache, value_cache=value_cache,
             key_scale=key_scale, value_scale=value_scale, block_tables=block_tables,
             seq_lens=seq_lens, new_lens=new_lens)


def run_attention(query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens,
                  words, scale, out_scale, max_seq_len, out, workspace, known=None):
    """Plan and launch a checked call (``known``: its :func:`_attention_plan`)."""
    slots, need, fields = known or _attention_plan(query, key_cache, key_scale, block_tables,
                                                   words, max_seq_len)
    index = query.device.index
    stream = _lib.raw_stream(index)
    if workspace is None:
        workspace = _lib.workspace_for(need, query, index, stream)
    elif workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous():
        raise ValueError(f"workspace_buffer must be contiguous and hold at least {need} bytes "
                         "for this batch")
    if out is None:
        out = torch.empty_like(query)
    _lib.launch_scaled(query, out, key_cache, value_cache, key_scale, value_scale, block_tables,
                       seq_lens, words, scale, out_scale, slots, workspace, stream, fields)
    return out


def _attention_plan(query, key_cache, key_scale, block_tables, words, max_seq_len):
    batch, q_len, hq, d = query.shape
    page, hkv = key_cache.shape[1], key_cache.shape[2]
    slots = _lib.plan_scaled(query.device.index, batch, hkv, max_seq_len,
                             block_tables.shape[1] * (page // 16))
    need = _lib.workspace_bytes(batch, q_len, hq, hkv, d, slots, 0)
    return slots, need, _lib.scaled_fields(query, key_cache, key_scale, block_tables, words)


def _check_attention(query, key_cache, value_cache, key_scale, value_scale, block_tables,
                     seq_lens, words, out, workspace_buffer):
    _check_cache(key_cache, value_cache, key_scale, value_scale)
    check_query(query, key_cache)
    check_batch(query.shape[0], block_tables, seq_lens)
    check_on(query.device, key_cache=key_cache, value_cache=value_cache, key_scale=key_scale,
             value_scale=value_scale, block_tables=block_tables, seq_lens=seq_lens, out=out,
             workspace_buffer=workspace_buffer, mask=words, query=query)
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype
                            or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor shaped and typed like query")


def paged_attention_scaled(query, key_cache, value_cache, key_scale, value_scale, block_tables,
                           seq_lens, max_seq_len: int = 0, scale: Optional[float] = None,
                           out_scale: float = 1.0, mask=None, out=None, workspace_buffer=None):
    """Small-q attention over a cache with block scales.

    ``query`` ``[B, Q, Hq, D]`` (fp16 or bf16; ``Q * Hq / Hkv <= 64``, 32 at head_dim 256):
    draft row ``i`` of sequence ``b`` sees the tokens before ``seq_lens[b] - Q`` and, of the
    last ``Q``, those up to its own or those ``mask`` names (the packed draft mask of
    :mod:`small_q_attention_amd.masks`). Rows that see no token are 0. ``max_seq_len`` > 0
    only sizes the call (0: the block table's width), and with it the last bits of a result
    may change; ``scale`` is the softmax scale (``None``: ``D ** -0.5``), ``out_scale``
    multiplies the output. V blocks of a scale under 2^-64 count as zeros; the V scales of
    what a row sees, those of zeros taken as 2^-64, may lie a factor of 2^100 apart. A token's
    probability times its V scale is rounded to fp16 in units of the row's largest: off by
    2^-11 of itself, or by 2^-25 of those units where it is small beside them.
    ``workspace_buffer``: a caller's buffer for the split partials; ``None`` takes one kept
    per host thread and stream, or, under graph capture, one of the graph's own. Returns ``out`` (``[B, Q, Hq, D]``).
    """
    if query.dim() != 4:
        raise ValueError("query must be a contiguous [B, Q, Hq, D] tensor")
    scale = check_softmax_scale(scale, query.shape[3])
    words = None if mask is None else as_words(mask, query.shape[0], query.shape[1])
    max_seq_len = min(max(int(max_seq_len), 0), 2**31 - 1)
    if _tracing():
        _check_attention(query, key_cache, value_cache, key_scale, value_scale, block_tables,
                         seq_lens, words, out, workspace_buffer)
        from . import _op  # noqa: F401  (registers the ops)

        res = torch.ops.sqa.paged_attention_scaled(
            query, key_cache, value_cache, key_scale, value_scale, block_tables, seq_lens, words,
            scale, float(out_scale), max_seq_len)
        return res if out is None else out.copy_(res)
    seen = (layout(query), layout(key_cache), layout(value_cache), layout(key_scale),
            layout(value_scale), layout(block_tables), layout(seq_lens), layout(words),
            layout(out), workspace_buffer is None or workspace_buffer.device, max_seq_len)
    known = _ATTENTIONS.get(seen)
    if known is None:
        _check_attention(query, key_cache, value_cache, key_scale, value_scale, block_tables,
                         seq_lens, words, out, workspace_buffer)
        known = _ATTENTIONS.keep(seen, on_device(query.device, _attention_plan, query, key_cache,
                                                 key_scale, block_tables, words, max_seq_len))
    check_aligned(16, query, key_cache, value_cache)
    return on_device(query.device, run_attention, query, key_cache, value_cache, key_scale,
                     value_scale, block_tables, seq_lens, words, scale, float(out_scale),
                     max_seq_len, out, workspace_buffer, known)


__all__ = ["append_scaled_kv", "paged_attention_scaled"]
