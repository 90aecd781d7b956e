"""ctypes binding of ``libsqa.so`` (C ABI in ``include/sqa.h``) and the torch custom op.

There is no fallback: if the library is missing or fails to load, every entry
point raises ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import functools
import struct
import threading
from pathlib import Path

from . import build as _build

_LOCK = threading.Lock()
_LIB = None

SQA_OK = 0

# (name, restype, argtypes) for every symbol include/sqa.h declares.
_C = ctypes
_SIGNATURES = [
    ("sqa_plan_splits", _C.c_int,
     [_C.c_int] * 9 + [_C.POINTER(_C.c_int), _C.POINTER(_C.c_int)]),
    ("sqa_workspace_bytes", _C.c_size_t, [_C.c_int] * 7),
    ("sqa_paged_mtp_attention", _C.c_int,
     [_C.c_void_p] * 7 + [_C.c_size_t] + [_C.c_int] * 5 + [_C.c_int64] + [_C.c_int] * 4
     + [_C.c_void_p, _C.c_void_p]),
    ("sqa_paged_mtp_attention_noalloc", _C.c_int,
     [_C.c_void_p] * 6 + [_C.c_int] * 5 + [_C.c_int64] + [_C.c_int] * 4 + [_C.c_void_p]),
    ("sqa_paged_attention", _C.c_int, [_C.c_void_p]),
    ("sqa_plan_scaled", _C.c_int, [_C.c_int] * 5 + [_C.POINTER(_C.c_int)]),
    ("sqa_paged_attention_scaled", _C.c_int, [_C.c_void_p, _C.c_void_p]),
    ("sqa_append_scaled", _C.c_int, [_C.c_void_p]),
    ("sqa_weights_workspace_bytes", _C.c_size_t, [_C.c_int] * 9),
    ("sqa_attention_weights", _C.c_int, [_C.c_void_p]),
    ("sqa_evict", _C.c_int, [_C.c_void_p]),
    ("sqa_device_cu_count", _C.c_int, [_C.c_int]),
    ("sqa_last_error", _C.c_char_p, []),
    ("sqa_version", _C.c_char_p, []),
]
EXPORTED = [name for name, _, _ in _SIGNATURES]


class KVCache(ctypes.Structure):
    """``sqa_kv_cache`` of include/sqa.h (strides in fp16 elements)."""

    _fields_ = [("k", _C.c_void_p), ("v", _C.c_void_p), ("num_pages", _C.c_int64),
                ("page_stride", _C.c_int64), ("token_stride", _C.c_int64),
                ("head_stride", _C.c_int64)]


class AttentionArgs(ctypes.Structure):
    """``sqa_attention_args`` of include/sqa.h."""

    _fields_ = [("struct_size", _C.c_size_t), ("query", _C.c_void_p), ("output", _C.c_void_p),
                ("kv", KVCache), ("block_tables", _C.c_void_p), ("seq_lens", _C.c_void_p),
                ("max_pages", _C.c_int), ("draft_mask", _C.c_void_p), ("mask_words", _C.c_int),
                ("scale", _C.c_float), ("out_scale", _C.c_float), ("batch", _C.c_int),
                ("q_len", _C.c_int), ("num_query_heads", _C.c_int), ("num_kv_heads", _C.c_int),
                ("head_dim", _C.c_int), ("page_size", _C.c_int), ("num_splits", _C.c_int),
                ("pages_per_split", _C.c_int), ("workspace", _C.c_void_p),
                ("workspace_bytes", _C.c_size_t), ("stream", _C.c_void_p),
                ("timing_events", _C.c_void_p), ("dtype", _C.c_int), ("kv_dtype", _C.c_int),
                ("flags", _C.c_int)]


class BlockScales(ctypes.Structure):
    """``sqa_block_scales`` of include/sqa.h (strides in floats)."""

    _fields_ = [("k", _C.c_void_p), ("v", _C.c_void_p), ("page_stride", _C.c_int64),
                ("head_stride", _C.c_int64)]


class AppendArgs(ctypes.Structure):
    """``sqa_append_args`` of include/sqa.h."""

    _fields_ = [("struct_size", _C.c_size_t), ("key", _C.c_void_p), ("value", _C.c_void_p),
                ("key_strides", _C.c_int64 * 3), ("value_strides", _C.c_int64 * 3),
                ("kv", KVCache), ("scales", BlockScales), ("block_tables", _C.c_void_p),
                ("seq_lens", _C.c_void_p), ("new_lens", _C.c_void_p), ("max_pages", _C.c_int),
                ("batch", _C.c_int), ("q_len", _C.c_int), ("num_kv_heads", _C.c_int),
                ("head_dim", _C.c_int), ("page_size", _C.c_int), ("dtype", _C.c_int),
                ("kv_dtype", _C.c_int), ("stream", _C.c_void_p)]


class WeightsArgs(ctypes.Structure):
    """``sqa_weights_args`` of include/sqa.h."""

    _fields_ = [("struct_size", _C.c_size_t), ("query", _C.c_void_p), ("kv", KVCache),
                ("k_scale", _C.c_void_p), ("scale_page_stride", _C.c_int64),
                ("scale_head_stride", _C.c_int64), ("block_tables", _C.c_void_p),
                ("seq_lens", _C.c_void_p), ("draft_mask", _C.c_void_p), ("weights", _C.c_void_p),
                ("weights_batch_stride", _C.c_int64), ("weights_head_stride", _C.c_int64),
                ("weights_width", _C.c_int), ("max_pages", _C.c_int), ("mask_words", _C.c_int),
                ("scale", _C.c_float), ("batch", _C.c_int), ("q_len", _C.c_int),
                ("num_query_heads", _C.c_int), ("num_kv_heads", _C.c_int),
                ("head_dim", _C.c_int), ("page_size", _C.c_int), ("max_seq_len", _C.c_int),
                ("dtype", _C.c_int), ("kv_dtype", _C.c_int), ("workspace", _C.c_void_p),
                ("workspace_bytes", _C.c_size_t), ("stream", _C.c_void_p)]


class EvictArgs(ctypes.Structure):
    """``sqa_evict_args`` of include/sqa.h."""

    _fields_ = [("struct_size", _C.c_size_t), ("weights", _C.c_void_p),
                ("weights_batch_stride", _C.c_int64), ("weights_head_stride", _C.c_int64),
                ("new_weights", _C.c_void_p), ("new_weights_batch_stride", _C.c_int64),
                ("new_weights_head_stride", _C.c_int64), ("kept", _C.c_void_p),
                ("seq_lens", _C.c_void_p), ("new_lens", _C.c_void_p), ("kv", KVCache),
                ("into", KVCache), ("scales", BlockScales), ("into_scales", BlockScales),
                ("block_tables", _C.c_void_p), ("new_tables", _C.c_void_p),
                ("weights_width", _C.c_int), ("new_weights_width", _C.c_int),
                ("max_pages", _C.c_int), ("new_max_pages", _C.c_int), ("budget", _C.c_int),
                ("sink", _C.c_int), ("recent", _C.c_int), ("batch", _C.c_int),
                ("num_kv_heads", _C.c_int), ("head_dim", _C.c_int), ("page_size", _C.c_int),
                ("kv_dtype", _C.c_int), ("stream", _C.c_void_p)]


# AttentionArgs as one packed record (native sizes and alignment, padded as C does).
_ARGS = struct.Struct("@N2P2P4q2PiPi2f8iPN2P3i0q")
assert _ARGS.size == ctypes.sizeof(AttentionArgs)
_SCALES = struct.Struct("@2P2q")
assert _SCALES.size == ctypes.sizeof(BlockScales)
_APPEND = struct.Struct("@N2P6q2P4q2P2q3P8iP0q")
assert _APPEND.size == ctypes.sizeof(AppendArgs)
_WEIGHTS = struct.Struct("@N3P4qP2q4P2q3if9iPNP0q")
assert _WEIGHTS.size == ctypes.sizeof(WeightsArgs)
_EVICT = struct.Struct("@NP2qP2q3P2P4q2P4q2P2q2P2q2P12iP0q")
assert _EVICT.size == ctypes.sizeof(EvictArgs)

DTYPE_F16, DTYPE_BF16, DTYPE_FP8_E4M3, DTYPE_INT8 = 0, 1, 2, 3
FLAG_ADAPTIVE_PAIRS = 1  # SQA_FLAG_ADAPTIVE_PAIRS


def library_path() -> Path:
    return _build.LIB_PATH


def load(verbose: bool = False, build_if_missing: bool = True):
    """Load ``libsqa.so``, building it first if it is missing or was built from other
    sources (the source hash stamped into the library differs from the hash of the
    sources beside it). With ``build_if_missing=False`` either case raises
    ``RuntimeError`` instead. ``verbose`` echoes the library path and the hipcc
    command that builds it, as the reference's loaders echo their JIT build
    (``cuda.py:31-36``)."""
    global _LIB
    if verbose:
        print(f"[sqa] {_build.LIB_PATH}; build command: {' '.join(_build.build_command())}",
              flush=True)
    with _LOCK:
        if _LIB is None:
            path = _build.LIB_PATH
            want = _build.source_hash()
            have = _build.built_hash(path) if path.exists() else None
            if have != want:
                if build_if_missing:
                    _build.build(verbose=verbose)
                elif not path.exists():
                    raise RuntimeError(f"{path} is not built; run small_q_attention_amd.build")
                elif have is not None:
                    raise RuntimeError(f"{path} is stale (built from sources {have}, sources "
                                       f"now {want}); run small_q_attention_amd.build")
                # An unstamped file: loading it below fails, or its version check does.
            try:
                lib = ctypes.CDLL(str(path))
            except OSError as exc:
                raise RuntimeError(f"cannot load {path}: {exc}") from exc
            for name, res, args in _SIGNATURES:
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            version = lib.sqa_version().decode(errors="replace")
            if f"sqa-src-hash:{want}" not in version:
                raise RuntimeError(f"{path} reports '{version}', not the sources' hash {want}; "
                                   "rebuild with small_q_attention_amd.build")
            _LIB = lib
        return _LIB


def last_error(lib) -> str:
    msg = lib.sqa_last_error()
    return msg.decode() if msg else "unknown error"


@functools.lru_cache(maxsize=4096)
def plan_splits(device_index: int, batch: int, q_len: int, num_query_heads: int,
                num_kv_heads: int, head_dim: int, max_seq_len: int, max_pages: int,
                chunk_keys: int):
    """``sqa_plan_splits`` -> ``(num_splits, pages_per_split)``; memoised (the plan is a
    pure function of its arguments and the device's CU count)."""
    lib = load()
    ns, pps = ctypes.c_int(0), ctypes.c_int(0)
    rc = lib.sqa_plan_splits(device_index, batch, q_len, num_query_heads, num_kv_heads,
                             head_dim, max_seq_len, max_pages, chunk_keys, ctypes.byref(ns),
                             ctypes.byref(pps))
    if rc != SQA_OK:
        raise RuntimeError(f"sqa_plan_splits failed: {last_error(lib)}")
    return ns.value, pps.value


@functools.lru_cache(maxsize=4096)
def workspace_bytes(batch: int, q_len: int, num_query_heads: int, num_kv_heads: int,
                    head_dim: int, num_splits: int, pages_per_split: int) -> int:
    """Workspace of a plan from :func:`plan_splits` (``pages_per_split`` 0 = balanced)."""
    return int(load().sqa_workspace_bytes(batch, q_len, num_query_heads, num_kv_heads, head_dim,
                                          num_splits, pages_per_split))


def raw_stream(device_index: int) -> int:
    """Handle of torch's current stream on ``device_index`` (a ``hipStream_t`` as int)."""
    import torch

    getter = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if getter is not None:
        return getter(device_index)
    return torch.cuda.current_stream(device_index).cuda_stream


def launch(query, key_cache, value_cache, block_tables, seq_lens, output, workspace,
           num_splits: int, pages_per_split: int, stream_handle: int, timing_events=None):
    """Call ``sqa_paged_mtp_attention`` on raw device pointers of torch tensors.

    The entry point reads fp16 elements through bare pointers, so any other
    element type (a bf16 or e4m3 cache: :func:`launch_general`) is refused here
    before the call; a 1-byte cache read as fp16 would run past its end."""
    for name, t in (("query", query), ("key_cache", key_cache), ("value_cache", value_cache),
                    ("output", output)):
        if str(t.dtype) != "torch.float16":
            raise TypeError(f"sqa_paged_mtp_attention takes fp16 tensors; {name} is {t.dtype} "
                            "(bf16 or e4m3 caches go through launch_general)")
    lib = _LIB if _LIB is not None else load()
    b, q_len, hq, d = query.shape
    ev = None
    if timing_events is not None:
        ev = (ctypes.c_void_p * 3)(*[ctypes.c_void_p(int(e)) for e in timing_events])
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    kshape = key_cache.shape
    rc = lib.sqa_paged_mtp_attention(
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
        block_tables.data_ptr(), seq_lens.data_ptr(), output.data_ptr(),
        ws_ptr, ws_bytes, b, q_len, hq, kshape[2], d,
        kshape[0], kshape[1], block_tables.shape[1],
        num_splits, pages_per_split, stream_handle, ev)
    if rc != SQA_OK:
        raise RuntimeError(f"sqa_paged_mtp_attention failed: {last_error(lib)}")


def launch_general(query, output, k_view, v_view, block_tables, seq_lens, draft_mask,
                   scale: float, out_scale: float, num_splits: int, pages_per_split: int,
                   workspace, stream_handle: int, timing_events=None, flags: int = 0):
    """Call ``sqa_paged_attention``. ``query``/``output``: contiguous ``[B, Q, Hq, D]``;
    ``k_view``/``v_view``: ``[num_pages, page, Hkv, D]`` views of equal strides with a
    contiguous head dimension (separate caches, or the K / V halves of an interleaved NHD
    or HND cache); ``draft_mask``: ``None`` (causal draft
    chain) or a contiguous 32-bit ``[B, Q, W]`` tensor of packed draft bits; ``flags``:
    0 or :data:`FLAG_ADAPTIVE_PAIRS`."""
    import torch

    lib = _LIB if _LIB is not None else load()
    b, q_len, hq, d = query.shape
    if k_view.dim() != 4 or v_view.shape != k_view.shape:
        raise ValueError("K and V views must both be [num_pages, page, Hkv, D]")
    strides = k_view.stride()
    if strides != v_view.stride() or strides[3] != 1:
        raise ValueError("K and V views must share strides with a contiguous head dimension")
    num_pages, page, hkv, _ = k_view.shape
    words, mask_words = (0, 0) if draft_mask is None else (draft_mask.data_ptr(),
                                                           draft_mask.shape[-1])
    ws, ws_bytes = (0, 0) if workspace is None else (
        workspace.data_ptr(), workspace.numel() * workspace.element_size())
    dtype = DTYPE_BF16 if query.dtype is torch.bfloat16 else DTYPE_F16
    kv_dtype = (DTYPE_FP8_E4M3
                if k_view.dtype is getattr(torch, "float8_e4m3fn", None) else dtype)
    ev = None
    if timing_events is not None:
        ev = (ctypes.c_void_p * 3)(*[ctypes.c_void_p(int(e)) for e in timing_events])
    # Every field at once: assigning them one by one took 4 us of a call.
    a = _ARGS.pack(
        _ARGS.size, query.data_ptr(), output.data_ptr(), k_view.data_ptr(), v_view.data_ptr(),
        num_pages, strides[0], strides[1], strides[2], block_tables.data_ptr(),
        seq_lens.data_ptr(), block_tables.shape[1], words, mask_words, scale, out_scale, b, q_len,
        hq, hkv, d, page, num_splits, pages_per_split, ws, ws_bytes, stream_handle or 0,
        0 if ev is None else ctypes.addressof(ev), dtype, kv_dtype, int(flags))
    rc = lib.sqa_paged_attention(a)
    if rc != SQA_OK:
        raise RuntimeError(f"sqa_paged_attention failed: {last_error(lib)}")


def dtype_code(dtype) -> int:
    """``SQA_DTYPE_*`` of a torch type."""
    return _DTYPE_CODES[str(dtype)]


_DTYPE_CODES = {"torch.float16": DTYPE_F16, "torch.bfloat16": DTYPE_BF16,
                "torch.float8_e4m3fn": DTYPE_FP8_E4M3, "torch.int8": DTYPE_INT8}


@functools.lru_cache(maxsize=4096)
def plan_scaled(device_index: int, batch: int, num_kv_heads: int, max_seq_len: int,
                max_pages: int) -> int:
    """``sqa_plan_scaled``: partial slots of a call over a cache with block scales."""
    lib = load()
    ns = ctypes.c_int(0)
    rc = lib.sqa_plan_scaled(device_index, batch, num_kv_heads, max_seq_len, max_pages,
                             ctypes.byref(ns))
    if rc != SQA_OK:
        raise RuntimeError(f"sqa_plan_scaled failed: {last_error(lib)}")
    return ns.value


def scaled_fields(query, k_view, k_scale, block_tables, draft_mask):
    """What of the arguments of ``sqa_paged_attention_scaled`` follows from the tensors'
    layouts."""
    b, q_len, hq, d = query.shape
    num_pages, page, hkv, _ = k_view.shape
    return ((num_pages, *k_view.stride()[:3]), block_tables.shape[1],
            0 if draft_mask is None else draft_mask.shape[-1], (b, q_len, hq, hkv, d, page),
            (dtype_code(query.dtype), dtype_code(k_view.dtype), 0), k_scale.stride())


def launch_scaled(query, output, k_view, v_view, k_scale, v_scale, block_tables, seq_lens,
                  draft_mask, scale: float, out_scale: float, num_splits: int, workspace,
                  stream_handle: int, fields=None):
    """Call ``sqa_paged_attention_scaled``: as :func:`launch_general`, over e4m3 or int8
    views with ``[num_pages, Hkv]`` float32 scales of equal strides (``fields`` from
    :func:`scaled_fields`)."""
    lib = _LIB if _LIB is not None else load()
    pool, max_pages, words, shape, types, scales = fields or scaled_fields(
        query, k_view, k_scale, block_tables, draft_mask)
    a = _ARGS.pack(
        _ARGS.size, query.data_ptr(), output.data_ptr(), k_view.data_ptr(), v_view.data_ptr(),
        *pool, block_tables.data_ptr(), seq_lens.data_ptr(), max_pages,
        0 if draft_mask is None else draft_mask.data_ptr(), words, scale, out_scale, *shape,
        num_splits, 0, workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        stream_handle or 0, 0, *types)
    rc = lib.sqa_paged_attention_scaled(
        a, _SCALES.pack(k_scale.data_ptr(), v_scale.data_ptr(), *scales))
    if rc != SQA_OK:
        raise RuntimeError(f"sqa_paged_attention_scaled failed: {last_error(lib)}")


def append_fields(key, value, k_view, k_scale, block_tables):
    """What of an ``sqa_append_args`` follows from the tensors' layouts (in its order, the
    pointers between)."""
    b, q_len, hkv, d = key.shape
    return ((*key.stride()[:3], *value.stride()[:3]), (k_view.shape[0], *k_view.stride()[:3]),
            k_scale.stride(), (block_tables.shape[1], b, q_len, hkv, d, k_view.shape[1],
                               dtype_code(key.dtype), dtype_code(k_view.dtype)))


def launch_append(key, value, k_view, v_view, k_scale, v_scale, block_tables, seq_lens, new_lens,
                  stream_handle: int, fields=None):
    """Call ``sqa_append_scaled`` (``key``/``value`` ``[B, Q, Hkv, D]``, their last dimension
    contiguous; views and scales as for :func:`launch_scaled`; ``fields`` from
    :func:`append_fields`)."""
    lib = _LIB if _LIB is not None else load()
    tokens, pool, scales, rest = fields or append_fields(key, value, k_view, k_scale, block_tables)
    rc = lib.sqa_append_scaled(_APPEND.pack(
        _APPEND.size, key.data_ptr(), value.data_ptr(), *tokens, k_view.data_ptr(),
        v_view.data_ptr(), *pool, k_scale.data_ptr(), v_scale.data_ptr(), *scales,
        block_tables.data_ptr(), seq_lens.data_ptr(),
        0 if new_lens is None else new_lens.data_ptr(), *rest, stream_handle or 0))
    if rc != SQA_OK:
        raise RuntimeError(f"sqa_append_scaled failed: {last_error(lib)}")


@functools.lru_cache(maxsize=4096)
def weights_workspace_bytes(device_index: int, batch: int, q_len: int, num_query_heads: int,
                            num_kv_heads: int, head_dim: int, max_seq_len: int, max_pages: int,
                            kv_dtype: int) -> int:
    """``sqa_weights_workspace_bytes`` (``max_pages``: 16-token pages)."""
    lib = load()
    need = lib.sqa_weights_workspace_bytes(device_index, batch, q_len, num_query_heads,
                                           num_kv_heads, head_dim, max_seq_len, max_pages,
                                           kv_dtype)
    if need == 0:
        raise RuntimeError(f"sqa_weights_workspace_bytes failed: {last_error(lib)}")
    return need


def weights_fields(query, k_view, k_scale, block_tables, draft_mask, weights, max_seq_len: int):
    """What of an ``sqa_weights_args`` follows from the tensors' layouts."""
    b, q_len, hq, d = query.shape
    return ((k_view.shape[0], *k_view.stride()[:3]), (0, 0) if k_scale is None
            else k_scale.stride(),
            (*weights.stride()[:2], weights.shape[2], block_tables.shape[1],
             0 if draft_mask is None else draft_mask.shape[-1]),
            (b, q_len, hq, k_view.shape[2], d, k_view.shape[1], max_seq_len,
             dtype_code(query.dtype), dtype_code(k_view.dtype)))


def launch_weights(query, k_view, k_scale, block_tables, seq_lens, draft_mask, weights,
                   scale: float, max_seq_len: int, workspace, stream_handle: int, fields=None):
    """Call ``sqa_attention_weights`` (``k_scale`` ``None``: none; ``weights`` ``[B, Hkv, T]``
    float32 with a contiguous last dimension; ``fields`` from :func:`weights_fields`)."""
    lib = _LIB if _LIB is not None else load()
    pool, scales, store, rest = fields or weights_fields(query, k_view, k_scale, block_tables,
                                                         draft_mask, weights, max_seq_len)
    rc = lib.sqa_attention_weights(_WEIGHTS.pack(
        _WEIGHTS.size, query.data_ptr(), k_view.data_ptr(), 0, *pool,
        0 if k_scale is None else k_scale.data_ptr(), *scales, block_tables.data_ptr(),
        seq_lens.data_ptr(), 0 if draft_mask is None else draft_mask.data_ptr(),
        weights.data_ptr(), *store, scale, *rest, workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), stream_handle or 0))
    if rc != SQA_OK:
        raise RuntimeError(f"sqa_attention_weights failed: {last_error(lib)}")


def evict_fields(weights, new_weights, source, into, block_tables, new_tables, budget: int,
                 sink: int, recent: int):
    """What of an ``sqa_evict_args`` follows from the tensors' layouts."""
    def strides(k, _v, ks, _vs):
        return (k.shape[0], *k.stride()[:3]), (0, 0) if ks is None else ks.stride()

    k = source[0]
    return (weights.stride()[:2], new_weights.stride()[:2], *strides(*source), *strides(*into),
            (weights.shape[2], new_weights.shape[2], block_tables.shape[1], new_tables.shape[1],
             budget, sink, recent, weights.shape[0], weights.shape[1], k.shape[3], k.shape[1],
             dtype_code(k.dtype)))


def launch_evict(weights, new_weights, kept, seq_lens, new_lens, source, into, block_tables,
                 new_tables, budget: int, sink: int, recent: int, stream_handle: int, fields=None):
    """Call ``sqa_evict``. ``source``, ``into``: (K view, V view, K scale, V scale), the
    scales ``None`` where the cache has none; ``fields`` from :func:`evict_fields`."""
    lib = _LIB if _LIB is not None else load()
    (w, nw, pool, scales, new_pool, new_scales, rest) = fields or evict_fields(
        weights, new_weights, source, into, block_tables, new_tables, budget, sink, recent)
    k, v, ks, vs = source
    k2, v2, ks2, vs2 = into
    sp = (0, 0) if ks is None else (ks.data_ptr(), vs.data_ptr())
    sp2 = (0, 0) if ks is None else (ks2.data_ptr(), vs2.data_ptr())
    rc = lib.sqa_evict(_EVICT.pack(
        _EVICT.size, weights.data_ptr(), *w, new_weights.data_ptr(), *nw, kept.data_ptr(),
        seq_lens.data_ptr(), new_lens.data_ptr(), k.data_ptr(), v.data_ptr(), *pool,
        k2.data_ptr(), v2.data_ptr(), *new_pool, *sp, *scales, *sp2, *new_scales,
        block_tables.data_ptr(), new_tables.data_ptr(), *rest, stream_handle or 0))
    if rc != SQA_OK:
        raise RuntimeError(f"sqa_evict failed: {last_error(lib)}")


def run(query, key_cache, value_cache, block_tables, seq_lens, num_splits: int,
        pages_per_split: int):
    """Allocate the output with torch's caching allocator, take a workspace from
    :func:`workspace_for`, and launch on the current stream of the query's device.
    Returns the output."""
    import torch

    out = torch.empty_like(query)
    b, q_len, hq, d = query.shape
    nbytes = workspace_bytes(b, q_len, hq, key_cache.shape[2], d, num_splits, pages_per_split)
    stream = raw_stream(query.device.index)
    ws = workspace_for(nbytes, query, query.device.index, stream) if nbytes else None
    if query.dtype == torch.float16:
        launch(query, key_cache, value_cache, block_tables, seq_lens, out, ws, num_splits,
               pages_per_split, stream)
    else:  # bf16: the general entry point carries the element type
        launch_general(query, out, key_cache, value_cache, block_tables, seq_lens, None,
                       query.shape[-1] ** -0.5, 1.0, num_splits, pages_per_split, ws, stream)
    return out


# Workspaces kept per host thread, device and stream for eager calls: a stream runs a
# thread's calls in order, so one buffer serves them all and the per-call allocation is
# saved. Each thread has its own: a call is two kernels, and between those of one thread
# another's may be launched on the same stream. Plans past WORKSPACE_CACHE_BYTES, and calls
# under graph capture (whose buffers belong to the graph's pool), allocate their own.
WORKSPACE_CACHE_BYTES = 64 << 20


class _Workspaces(threading.local):
    def __init__(self):
        self.of = {}


_WORKSPACES = _Workspaces()
_CUDA_STATE = None  # (current device, current stream capturing): torch's own query functions


def _cuda_state(torch):
    """The functions behind ``torch.cuda.current_device`` and
    ``torch.cuda.is_current_stream_capturing`` without their per-call
    initialisation checks (callers hold a CUDA tensor, so CUDA is initialised);
    the public ones where this torch lacks them."""
    global _CUDA_STATE
    if _CUDA_STATE is None:
        c = torch._C
        _CUDA_STATE = (getattr(c, "_cuda_getDevice", None) or torch.cuda.current_device,
                       getattr(c, "_cuda_isCurrentStreamCapturing", None)
                       or torch.cuda.is_current_stream_capturing)
    return _CUDA_STATE


def workspace_for(nbytes: int, like, device_index: int, stream_handle: int):
    """A workspace of at least ``nbytes`` for a call on ``stream_handle`` (``like``: a
    tensor on the call's device)."""
    import torch

    current_device, capturing = _CUDA_STATE or _cuda_state(torch)
    # The capture check reads the current device's stream: the cache serves only
    # calls on that device.
    if nbytes > WORKSPACE_CACHE_BYTES or device_index != current_device() or capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    key = (device_index, stream_handle)
    mine = _WORKSPACES.of
    ws = mine.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=like.device)
        mine[key] = ws
    return ws


def run_fp16(query, key_cache, value_cache, block_tables, seq_lens, batch: int, q_len: int,
             num_query_heads: int, num_kv_heads: int, num_pages: int, page_size: int,
             max_pages: int, num_splits: int, pages_per_split: int, device_index: int):
    """:func:`run` for the fp16, head-dim-128 call whose shapes the caller has already
    checked and unpacked: the same allocation and launch with fewer Python steps."""
    import torch

    out = torch.empty_like(query)
    nbytes = workspace_bytes(batch, q_len, num_query_heads, num_kv_heads, 128, num_splits,
                             pages_per_split)
    stream = raw_stream(device_index)
    ws = workspace_for(nbytes, query, device_index, stream) if nbytes else None
    rc = _LIB.sqa_paged_mtp_attention(
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
        block_tables.data_ptr(), seq_lens.data_ptr(), out.data_ptr(),
        ws.data_ptr() if ws is not None else None, nbytes, batch, q_len, num_query_heads,
        num_kv_heads, 128, num_pages, page_size, max_pages, num_splits, pages_per_split,
        stream, None)
    if rc != SQA_OK:
        raise RuntimeError(f"sqa_paged_mtp_attention failed: {last_error(_LIB)}")
    return out


def custom_op():
    """The ``sqa::paged_mtp_attention`` torch custom op (registered on first use)."""
    from . import _op

    return _op.paged_mtp_attention
