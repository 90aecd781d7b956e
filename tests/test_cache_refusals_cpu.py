"""What the operators around the paged cache refuse, checked without a GPU: the Python
entry points' ValueErrors, the C ABI's status codes, the traced ops' registration."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd import _lib, _op, build, eviction, scaled_cache  # noqa: E402,F401

F16, BF16, E4M3, INT8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn, torch.int8


def _zeros(*shape, dtype=torch.float32):
    x = torch.zeros(*shape, dtype=torch.uint8 if dtype is E4M3 else dtype)
    return x.view(E4M3) if dtype is E4M3 else x


def _base(kv=E4M3, dtype=F16, b=2, q=3, hq=8, hkv=2, d=64, pages=6, page=16, width=4):
    return dict(
        key=_zeros(b, q, hkv, d, dtype=dtype), value=_zeros(b, q, hkv, d, dtype=dtype),
        query=_zeros(b, q, hq, d, dtype=dtype),
        key_cache=_zeros(pages, page, hkv, d, dtype=kv),
        value_cache=_zeros(pages, page, hkv, d, dtype=kv),
        key_scale=torch.ones(pages, hkv), value_scale=torch.ones(pages, hkv),
        block_tables=torch.zeros(b, width, dtype=torch.int32),
        seq_lens=torch.ones(b, dtype=torch.int32), weights=torch.zeros(b, hkv, 64),
        new_block_tables=torch.zeros(b, 2, dtype=torch.int32))


def _append(a, **kw):
    return scaled_cache.append_scaled_kv(
        a["key"], a["value"], a["key_cache"], a["value_cache"], a["key_scale"], a["value_scale"],
        a["block_tables"], a["seq_lens"], **kw)


def _attend(a, **kw):
    return scaled_cache.paged_attention_scaled(
        a["query"], a["key_cache"], a["value_cache"], a["key_scale"], a["value_scale"],
        a["block_tables"], a["seq_lens"], **kw)


def _weigh(a, **kw):
    kw.setdefault("key_scale", a["key_scale"])
    return eviction.accumulate_attention_weights(a["query"], a["key_cache"], a["block_tables"],
                                                 a["seq_lens"], a["weights"], **kw)


def _evict(a, **kw):
    kw.setdefault("budget", 20)
    kw.setdefault("key_scale", a["key_scale"])
    kw.setdefault("value_scale", a["value_scale"])
    return eviction.evict_by_weight(a["weights"], a["key_cache"], a["value_cache"],
                                    a["block_tables"], a["seq_lens"], a["new_block_tables"], **kw)


CALLS = {"append": _append, "attend": _attend, "weigh": _weigh, "evict": _evict}


@pytest.mark.parametrize("call", CALLS)
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="GPU"):
        CALLS[call](_base())


@pytest.mark.parametrize("call,change,match", [
    # caches
    ("append", dict(key_cache=_zeros(6, 16, 2, 64, dtype=F16)), "float8|int8"),
    ("attend", dict(key_cache=_zeros(6, 16, 2, 64, dtype=BF16)), "float8|int8"),
    ("attend", dict(value_cache=_zeros(6, 16, 2, 64, dtype=INT8)), "match"),
    ("attend", dict(value_cache=_zeros(7, 16, 2, 64, dtype=E4M3)), "match"),
    ("append", dict(key_cache=_zeros(6, 24, 2, 64, dtype=E4M3)), "page_size"),
    ("weigh", dict(key_cache=_zeros(6, 8, 2, 64, dtype=E4M3)), "page_size"),
    ("weigh", dict(key_cache=_zeros(6, 16, 2, 96, dtype=E4M3)), "head_dim"),
    ("attend", dict(key_cache=_zeros(0, 16, 2, 64, dtype=E4M3)), "empty"),
    ("attend", dict(key_cache=_zeros(6, 16, 2, 128, dtype=E4M3)[..., ::2]), "contiguous head"),
    ("evict", dict(key_cache=_zeros(6, 16, 2, 72, dtype=E4M3)[..., :64],
                   value_cache=_zeros(6, 16, 2, 72, dtype=E4M3)[..., :64]), "16 bytes"),
    ("evict", dict(key_cache=torch.zeros(6, 16, 2, 64), value_cache=torch.zeros(6, 16, 2, 64)),
     "hold"),
    # scales
    ("append", dict(key_scale=torch.ones(6, 2, dtype=torch.float64)), "float32"),
    ("attend", dict(value_scale=torch.ones(6, 3)), "float32"),
    ("attend", dict(value_scale=torch.ones(2, 6).t()), "match"),
    ("evict", dict(value_scale=None), "together"),
    ("weigh", dict(key_cache=_zeros(6, 16, 2, 64, dtype=F16)), "scales belong"),
    ("weigh", dict(key_cache=_zeros(6, 16, 2, 64, dtype=INT8), key_scale=None), "int8"),
    ("weigh", dict(key_cache=_zeros(6, 16, 2, 64, dtype=BF16), key_scale=None), "query's type"),
    # tables and lengths
    ("append", dict(block_tables=torch.zeros(2, 4, dtype=torch.int64)), "int32"),
    ("attend", dict(block_tables=torch.zeros(3, 4, dtype=torch.int32)), "contiguous"),
    ("attend", dict(block_tables=torch.zeros(4, 2, dtype=torch.int32).t()), "contiguous"),
    ("weigh", dict(seq_lens=torch.ones(3, dtype=torch.int32)), "seq_lens"),
    ("evict", dict(new_block_tables=torch.zeros(2, 2, dtype=torch.int64)), "int32"),
    ("evict", dict(new_block_tables=torch.zeros(2, 1, dtype=torch.int32)), "pages for budget"),
    # queries and tokens
    ("attend", dict(query=torch.zeros(2, 3, 8, 64)), "float16 or bfloat16"),
    ("attend", dict(query=_zeros(2, 3, 8, 128, dtype=F16)), "head_dim"),
    ("attend", dict(query=_zeros(2, 3, 7, 64, dtype=F16)), "multiple"),
    ("attend", dict(query=_zeros(2, 17, 8, 64, dtype=F16)), "at most 64"),
    ("weigh", dict(query=_zeros(2, 17, 8, 64, dtype=F16)), "at most 64"),
    ("weigh", dict(query=_zeros(2, 0, 8, 64, dtype=F16)), "contiguous"),
    ("attend", dict(query=_zeros(6, 8, 64, dtype=F16)), "contiguous"),
    ("append", dict(key=torch.zeros(2, 3, 2, 64)), "float16 or bfloat16"),
    ("append", dict(value=_zeros(2, 3, 2, 64, dtype=BF16)), "float16 or bfloat16"),
    ("append", dict(value=_zeros(2, 4, 2, 64, dtype=F16)), "one shape"),
    ("append", dict(key=_zeros(2, 3, 1, 64, dtype=F16), value=_zeros(2, 3, 1, 64, dtype=F16)),
     "kv heads"),
    ("append", dict(key=_zeros(2, 3, 2, 68, dtype=F16)[..., :64]), "multiples of 8"),
    ("append", dict(key_cache=_zeros(1, 16, 2, 64, dtype=E4M3).expand(6, -1, -1, -1),
                    value_cache=_zeros(1, 16, 2, 64, dtype=E4M3).expand(6, -1, -1, -1)), "expanded"),
    ("append", dict(key_scale=torch.ones(1, 2).expand(6, 2),
                    value_scale=torch.ones(1, 2).expand(6, 2)), "expanded"),
    # weights
    ("weigh", dict(weights=torch.zeros(1, 2, 64).expand(2, -1, -1)), "expanded"),
    ("weigh", dict(weights=torch.zeros(2, 2, 64, dtype=torch.float64)), "float32"),
    ("weigh", dict(weights=torch.zeros(2, 3, 64)), "float32"),
    ("evict", dict(weights=torch.zeros(2, 64, 2).transpose(1, 2)), "contiguous"),
])
def test_tensors_outside_the_contract(call, change, match):
    a = _base()
    a.update(change)
    with pytest.raises(ValueError, match=match):
        CALLS[call](a)


@pytest.mark.parametrize("call,kw,match", [
    ("append", dict(new_lens=torch.ones(3, dtype=torch.int32)), "new_lens"),
    ("append", dict(new_lens=torch.ones(2, dtype=torch.int64)), "new_lens"),
    ("attend", dict(scale=0.0), "positive"),
    ("attend", dict(scale=float("nan")), "positive"),
    ("attend", dict(mask=torch.zeros(2, 4, 1, dtype=torch.int32)), "mask"),
    ("weigh", dict(scale=-1.0), "positive"),
    ("weigh", dict(scale=float("inf")), "positive"),
    ("evict", dict(budget=0), "budget"),
    ("evict", dict(sink=-1), "budget"),
    ("evict", dict(sink=11, recent=10), "budget"),
    ("evict", dict(into=(1,)), None),
    ("evict", dict(new_weights=torch.zeros(2, 2, 19)), "new_weights"),
])
def test_arguments_outside_the_contract(call, kw, match):
    a = _base()
    if "into" in kw:
        kw = dict(into=(a["key_cache"], a["value_cache"], a["key_scale"]))
    with pytest.raises(ValueError, match=match):
        CALLS[call](a, **kw)


def test_more_rows_than_head_dim_256_carries():
    a = _base(d=256, q=9)
    for call in ("attend", "weigh"):
        with pytest.raises(ValueError, match="at most 32"):
            CALLS[call](a)


def test_into_must_be_like_the_cache():
    a = _base()
    wide = (_zeros(6, 32, 2, 64, dtype=E4M3),) * 2 + (a["key_scale"],) * 2
    with pytest.raises(ValueError, match="page size"):
        _evict(a, into=wide)
    with pytest.raises(ValueError, match="scales where"):
        _evict(a, into=(a["key_cache"], a["value_cache"]))


# ----- the C ABI -----

INVALID, UNSUPPORTED = 1, 2


@pytest.fixture(scope="module")
def lib():
    if build.is_stale():
        build.build()
    return _lib.load()


def _fill(struct, **kw):
    s = struct()
    s.struct_size = ctypes.sizeof(struct)
    for k, v in kw.items():
        at = s
        *path, last = k.split("__")
        for p in path:
            at = getattr(at, p)
        setattr(at, last, v)
    return s


def _scales(**kw):
    return _fill_plain(_lib.BlockScales, **{**dict(k=4096, v=4096, page_stride=2, head_stride=1),
                                            **kw})


def _fill_plain(struct, **kw):
    s = struct()
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _attention_args(**kw):
    return _fill(_lib.AttentionArgs, **{**dict(
        query=4096, output=4096, kv__k=4096, kv__v=4096, kv__num_pages=6, kv__page_stride=2048,
        kv__token_stride=128, kv__head_stride=64, block_tables=4096, seq_lens=4096, max_pages=4,
        scale=0.125, out_scale=1.0, batch=2, q_len=3, num_query_heads=8, num_kv_heads=2,
        head_dim=64, page_size=16, num_splits=2, pages_per_split=0, workspace=4096,
        workspace_bytes=1 << 20, dtype=0, kv_dtype=2), **kw})


@pytest.mark.parametrize("change,status", [
    (dict(struct_size=8), INVALID), (dict(query=None), INVALID), (dict(query=4104), INVALID),
    (dict(batch=0), INVALID), (dict(kv__num_pages=0), INVALID), (dict(kv__num_pages=1 << 31), INVALID),
    (dict(num_query_heads=7), INVALID), (dict(q_len=17), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED),
    (dict(page_size=48), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED), (dict(kv_dtype=0), UNSUPPORTED),
    (dict(kv_dtype=4), UNSUPPORTED), (dict(kv__token_stride=-8), INVALID),
    (dict(kv__token_stride=4), INVALID), (dict(kv__page_stride=1 << 41), INVALID),
    (dict(kv__token_stride=1 << 29), INVALID), (dict(scale=0.0), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(out_scale=float("nan")), INVALID),
    (dict(flags=1), INVALID), (dict(pages_per_split=4), INVALID), (dict(num_splits=1), INVALID),
    (dict(max_pages=1 << 27), INVALID), (dict(draft_mask=4096, mask_words=0), INVALID),
    (dict(workspace=None), 3), (dict(workspace_bytes=100), 3), (dict(workspace=4100), 3),
    (dict(num_splits=1 << 30, workspace_bytes=1 << 62), INVALID),
])
def test_attention_status(lib, change, status):
    a, s = _attention_args(**change), _scales()
    assert lib.sqa_paged_attention_scaled(ctypes.byref(a), ctypes.byref(s)) == status
    assert lib.sqa_last_error()


@pytest.mark.parametrize("change", [dict(k=None), dict(v=None), dict(k=4098), dict(page_stride=-1),
                                    dict(head_stride=-1), dict(head_stride=1 << 31)])
def test_scale_status(lib, change):
    a, s = _attention_args(), _scales(**change)
    assert lib.sqa_paged_attention_scaled(ctypes.byref(a), ctypes.byref(s)) == INVALID
    assert lib.sqa_paged_attention_scaled(None, ctypes.byref(s)) == INVALID
    assert lib.sqa_paged_attention_scaled(ctypes.byref(a), None) == INVALID


@pytest.mark.parametrize("change,status", [
    (dict(struct_size=8), INVALID), (dict(key=None), INVALID), (dict(key=4104), INVALID),
    (dict(q_len=0), INVALID), (dict(dtype=3), UNSUPPORTED), (dict(kv_dtype=1), UNSUPPORTED),
    (dict(scales__k=None), INVALID), (dict(new_lens=4097), INVALID), (dict(page_size=8), UNSUPPORTED),
    (dict(kv__v=4100), INVALID), (dict(max_pages=0), INVALID), (dict(head_dim=32), UNSUPPORTED),
])
def test_append_status(lib, change, status):
    a = _fill(_lib.AppendArgs, **{**dict(
        key=4096, value=4096, kv__k=4096, kv__v=4096, kv__num_pages=6, kv__page_stride=2048,
        kv__token_stride=128, kv__head_stride=64, scales__k=4096, scales__v=4096,
        scales__page_stride=2, scales__head_stride=1, block_tables=4096, seq_lens=4096, max_pages=4,
        batch=2, q_len=3, num_kv_heads=2, head_dim=64, page_size=16, dtype=0, kv_dtype=2), **change})
    a.key_strides[:] = a.value_strides[:] = (384, 128, 64)
    assert lib.sqa_append_scaled(ctypes.byref(a)) == status
    a.struct_size = ctypes.sizeof(a)
    a.key_strides[1] = 4
    assert lib.sqa_append_scaled(ctypes.byref(a)) in (INVALID, UNSUPPORTED)
    assert lib.sqa_append_scaled(None) == INVALID


@pytest.mark.parametrize("change,status", [
    (dict(struct_size=8), INVALID), (dict(weights=None), INVALID), (dict(weights=4097), INVALID),
    (dict(kv_dtype=1), UNSUPPORTED), (dict(k_scale=4096, kv_dtype=0), INVALID),
    (dict(kv_dtype=3), INVALID), (dict(scale=-1.0), INVALID), (dict(weights_width=0), INVALID),
    (dict(weights_head_stride=-1), INVALID), (dict(q_len=17), UNSUPPORTED),
])
def test_weights_status(lib, change, status):
    a = _fill(_lib.WeightsArgs, **{**dict(
        query=4096, kv__k=4096, kv__num_pages=6, kv__page_stride=2048, kv__token_stride=128,
        kv__head_stride=64, block_tables=4096, seq_lens=4096, weights=4096,
        weights_batch_stride=128, weights_head_stride=64, weights_width=64, max_pages=4, scale=0.1,
        batch=2, q_len=3, num_query_heads=8, num_kv_heads=2, head_dim=64, page_size=16, dtype=0,
        kv_dtype=0, workspace=4096, workspace_bytes=1 << 20), **change})
    assert lib.sqa_attention_weights(ctypes.byref(a)) == status
    assert lib.sqa_attention_weights(None) == INVALID


@pytest.mark.parametrize("change,status", [
    (dict(struct_size=8), INVALID), (dict(kept=None), INVALID), (dict(kept=4097), INVALID),
    (dict(budget=0), INVALID), (dict(budget=33), INVALID), (dict(sink=30, recent=3), INVALID),
    (dict(new_weights_width=19), INVALID), (dict(weights_width=0), INVALID),
    (dict(kv_dtype=4), UNSUPPORTED), (dict(kv_dtype=3), INVALID), (dict(scales__k=4096), INVALID),
    (dict(kv_dtype=2, kv__head_stride=72), INVALID), (dict(into__num_pages=0), INVALID),
    (dict(new_max_pages=0), INVALID), (dict(into__k=4104), INVALID),
])
def test_evict_status(lib, change, status):
    pool = dict(k=4096, v=4096, num_pages=6, page_stride=2048, token_stride=128, head_stride=64)
    a = _fill(_lib.EvictArgs, **{**dict(
        weights=4096, weights_batch_stride=128, weights_head_stride=64, new_weights=4096,
        new_weights_batch_stride=40, new_weights_head_stride=20, kept=4096, seq_lens=4096,
        new_lens=4096, block_tables=4096, new_tables=4096, weights_width=64, new_weights_width=20,
        max_pages=4, new_max_pages=2, budget=20, sink=2, recent=3, batch=2, num_kv_heads=2,
        head_dim=64, page_size=16, kv_dtype=0, **{f"kv__{k}": v for k, v in pool.items()},
        **{f"into__{k}": v for k, v in pool.items()}), **change})
    assert lib.sqa_evict(ctypes.byref(a)) == status
    assert lib.sqa_evict(None) == INVALID


@pytest.mark.parametrize("change", [dict(kv__v=4096), dict(scales__v=4096)],
                         ids=["caches", "scales"])
def test_append_needs_a_cache_each_for_keys_and_values(lib, change):
    a = _fill(_lib.AppendArgs, **{**dict(
        key=4096, value=4096, kv__k=4096, kv__v=1 << 20, kv__num_pages=6, kv__page_stride=2048,
        kv__token_stride=128, kv__head_stride=64, scales__k=4096, scales__v=8192,
        scales__page_stride=2, scales__head_stride=1, block_tables=4096, seq_lens=4096, max_pages=4,
        batch=2, q_len=3, num_kv_heads=2, head_dim=64, page_size=16, dtype=0, kv_dtype=2), **change})
    a.key_strides[:] = a.value_strides[:] = (384, 128, 64)
    assert lib.sqa_append_scaled(ctypes.byref(a)) == INVALID
    assert b"own cache" in lib.sqa_last_error()


@pytest.mark.parametrize("change", [dict(into__v=4096), dict(into_scales__v=4096)],
                         ids=["caches", "scales"])
def test_evict_needs_a_cache_each_for_keys_and_values(lib, change):
    pool = dict(k=4096, v=1 << 20, num_pages=6, page_stride=2048, token_stride=128, head_stride=64)
    sc = dict(k=4096, v=8192, page_stride=2, head_stride=1)
    a = _fill(_lib.EvictArgs, **{**dict(
        weights=4096, weights_batch_stride=128, weights_head_stride=64, new_weights=4096,
        new_weights_batch_stride=40, new_weights_head_stride=20, kept=4096, seq_lens=4096,
        new_lens=4096, block_tables=4096, new_tables=4096, weights_width=64, new_weights_width=20,
        max_pages=4, new_max_pages=2, budget=20, sink=2, recent=3, batch=2, num_kv_heads=2,
        head_dim=64, page_size=16, kv_dtype=2, **{f"kv__{k}": v for k, v in pool.items()},
        **{f"into__{k}": v for k, v in pool.items()}, **{f"scales__{k}": v for k, v in sc.items()},
        **{f"into_scales__{k}": v for k, v in sc.items()}), **change})
    assert lib.sqa_evict(ctypes.byref(a)) == INVALID
    assert b"own cache" in lib.sqa_last_error()


def _evict_args(**kw):
    """Arguments of an sqa_evict call with nothing to refuse."""
    pool = dict(k=1 << 16, v=1 << 17, num_pages=6, page_stride=2048, token_stride=128, head_stride=64)
    sc = dict(k=1 << 18, v=1 << 19, page_stride=2, head_stride=1)
    return _fill(_lib.EvictArgs, **{**dict(
        weights=1 << 20, weights_batch_stride=128, weights_head_stride=64, new_weights=2 << 20,
        new_weights_batch_stride=40, new_weights_head_stride=20, kept=3 << 20, seq_lens=4 << 20,
        new_lens=5 << 20, block_tables=6 << 20, new_tables=7 << 20, weights_width=64,
        new_weights_width=20, max_pages=4, new_max_pages=2, budget=20, sink=2, recent=3, batch=2,
        num_kv_heads=2, head_dim=64, page_size=16, kv_dtype=2,
        **{f"kv__{k}": v for k, v in pool.items()}, **{f"into__{k}": v for k, v in pool.items()},
        **{f"scales__{k}": v for k, v in sc.items()},
        **{f"into_scales__{k}": v for k, v in sc.items()}), **kw})


# No test below reaches a launch where there is a GPU: made-up pointers must not get there.
without_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="passes made-up pointers on")


@without_gpu
@pytest.mark.parametrize("by", [0, 4, -4])
def test_evict_lengths_are_not_written_over(lib, by):
    a = _evict_args(new_lens=(4 << 20) + by)
    assert lib.sqa_evict(ctypes.byref(a)) == INVALID
    assert b"new_lens must not overlap" in lib.sqa_last_error()
    a = _evict_args(new_lens=(4 << 20) + 2 * by + (8 if by == 0 else 0))  # beside them
    assert lib.sqa_evict(ctypes.byref(a)) == 4


def _append_args(**kw):
    """Arguments of an sqa_append_scaled call with nothing to refuse."""
    a = _fill(_lib.AppendArgs, **{**dict(
        key=1 << 16, value=1 << 17, kv__k=1 << 18, kv__v=1 << 19, kv__num_pages=6,
        kv__page_stride=2048, kv__token_stride=128, kv__head_stride=64, scales__k=1 << 20,
        scales__v=2 << 20, scales__page_stride=2, scales__head_stride=1, block_tables=3 << 20,
        seq_lens=4 << 20, max_pages=4, batch=2, q_len=3, num_kv_heads=2, head_dim=64, page_size=16,
        dtype=0, kv_dtype=2), **{k: v for k, v in kw.items() if not k.endswith("_strides")}})
    a.key_strides[:] = kw.get("key_strides", (384, 128, 64))
    a.value_strides[:] = kw.get("value_strides", (384, 128, 64))
    return a


# Each row changes one thing of a call that is otherwise taken, so its message names the
# check it is about.

@without_gpu
@pytest.mark.parametrize("change,status,message", [
    (dict(), 4, ""),
    (dict(struct_size=8), INVALID, "struct_size"), (dict(key=None), INVALID, "null tensor"),
    (dict(value=None), INVALID, "null tensor"), (dict(kv__v=None), INVALID, "null tensor"),
    (dict(block_tables=None), INVALID, "null tensor"), (dict(seq_lens=None), INVALID, "null tensor"),
    (dict(key=(1 << 16) + 8), INVALID, "16-byte"), (dict(value=(1 << 17) + 2), INVALID, "16-byte"),
    (dict(batch=0), INVALID, "batch"), (dict(q_len=0), INVALID, "q_len"),
    (dict(dtype=3), UNSUPPORTED, "dtype"), (dict(kv_dtype=1), UNSUPPORTED, "kv_dtype"),
    (dict(scales__k=None), INVALID, "null scale"), (dict(scales__v=None), INVALID, "null scale"),
    (dict(scales__k=(1 << 20) + 2), INVALID, "scales must be 4-byte"),
    (dict(scales__page_stride=-1), INVALID, "scale strides"),
    (dict(scales__head_stride=1 << 30), INVALID, "scale strides"),
    (dict(new_lens=4097), INVALID, "new_lens"), (dict(seq_lens=4098), INVALID, "seq_lens"),
    (dict(block_tables=4098), INVALID, "block_tables"), (dict(page_size=8), UNSUPPORTED, "page_size"),
    (dict(kv__v=(1 << 19) + 4), INVALID, "base pointers"), (dict(max_pages=0), INVALID, "empty"),
    (dict(kv__num_pages=1 << 31), INVALID, "32 bits"), (dict(max_pages=1 << 26), INVALID, "2^30"),
    (dict(head_dim=32), UNSUPPORTED, "head_dim"), (dict(kv__page_stride=-8), INVALID, "cache strides"),
    (dict(kv__head_stride=4), INVALID, "cache strides"),
    (dict(kv__token_stride=1 << 31), INVALID, "too large"),
    (dict(kv__token_stride=1 << 29), INVALID, "2 GiB"),
    (dict(key_strides=(384, 4, 64)), INVALID, "key and value strides"),
    (dict(value_strides=(384, 128, -64)), INVALID, "key and value strides"),
    (dict(kv__v=1 << 18), INVALID, "own cache"), (dict(scales__v=1 << 20), INVALID, "own cache"),
    (dict(batch=1 << 15, q_len=1 << 20, num_kv_heads=1 << 14, max_pages=1 << 14,
          kv__head_stride=64), INVALID, "grid"),
])
def test_each_refusal_of_an_append(lib, change, status, message):
    assert lib.sqa_append_scaled(ctypes.byref(_append_args(**change))) == status
    assert message in lib.sqa_last_error().decode()


@without_gpu
@pytest.mark.parametrize("change,status,message", [
    (dict(), 4, ""),
    (dict(struct_size=8), INVALID, "struct_size"), (dict(weights=None), INVALID, "null tensor"),
    (dict(new_weights=None), INVALID, "null tensor"), (dict(kept=None), INVALID, "null tensor"),
    (dict(new_lens=None), INVALID, "null tensor"), (dict(new_tables=None), INVALID, "null tensor"),
    (dict(into__v=None), INVALID, "null tensor"),
    (dict(kept=(3 << 20) + 1), INVALID, "4-byte aligned"),
    (dict(weights=(1 << 20) + 2), INVALID, "4-byte aligned"),
    (dict(new_tables=(7 << 20) + 2), INVALID, "4-byte aligned"),
    (dict(batch=0), INVALID, "batch"), (dict(kv__num_pages=0), INVALID, "empty"),
    (dict(into__num_pages=0), INVALID, "empty"), (dict(max_pages=0), INVALID, "empty"),
    (dict(new_max_pages=0), INVALID, "empty"), (dict(head_dim=96), UNSUPPORTED, "head_dim"),
    (dict(page_size=24), UNSUPPORTED, "page_size"), (dict(kv_dtype=4), UNSUPPORTED, "kv_dtype"),
    (dict(budget=0), INVALID, "budget must be positive"), (dict(sink=-1), INVALID, "budget must be"),
    (dict(recent=-1), INVALID, "budget must be"), (dict(sink=18), INVALID, "budget must be"),
    (dict(budget=33, new_weights_width=33), INVALID, "new_tables rows hold"),
    (dict(new_weights_width=19), INVALID, "new_weights hold"),
    (dict(weights_width=0), INVALID, "must not be empty"),
    (dict(weights_head_stride=-1), INVALID, "not be negative"),
    (dict(new_weights_batch_stride=-1), INVALID, "not be negative"),
    (dict(kv_dtype=3, scales__k=None), INVALID, "int8 caches need scales"),
    (dict(kv_dtype=0), INVALID, "scales belong"), (dict(scales__v=None), INVALID, "null scale"),
    (dict(into_scales__k=None), INVALID, "null scale"),
    (dict(into_scales__head_stride=-1), INVALID, "scale strides"),
    (dict(kv__head_stride=72), INVALID, "16 bytes"), (dict(into__page_stride=2056), INVALID, "16 bytes"),
    (dict(kv__token_stride=4), INVALID, "multiples of 8"),
    (dict(into__k=(1 << 16) + 4), INVALID, "base pointers"),
    (dict(into__v=1 << 16), INVALID, "own cache"), (dict(into_scales__v=1 << 18), INVALID, "own cache"),
    (dict(new_lens=4 << 20), INVALID, "overlap"),
    (dict(batch=1 << 16, num_kv_heads=1 << 16, max_pages=1, new_max_pages=2), INVALID, "grid"),
])
def test_each_refusal_of_an_eviction(lib, change, status, message):
    assert lib.sqa_evict(ctypes.byref(_evict_args(**change))) == status
    assert message in lib.sqa_last_error().decode()


# ----- the traced ops -----

@pytest.mark.parametrize("name,writes", [
    ("paged_attention_scaled", set()),
    ("append_scaled_kv", {"key_cache", "value_cache", "key_scale", "value_scale"}),
    ("accumulate_attention_weights", {"weights"}),
    ("evict_by_weight", {"new_key_cache", "new_value_cache", "new_key_scale", "new_value_scale",
                         "new_weights", "new_lens", "kept"}),
])
def test_ops_say_what_they_write(name, writes):
    op = getattr(torch.ops.sqa, name).default
    assert {a.name for a in op._schema.arguments
            if a.alias_info is not None and a.alias_info.is_write} == writes


def test_fake_attention_shapes_its_output():
    m = {k: v.to("meta") if v.dtype is not E4M3 else torch.empty(v.shape, dtype=E4M3, device="meta")
         for k, v in _base().items()}
    out = torch.ops.sqa.paged_attention_scaled(
        m["query"], m["key_cache"], m["value_cache"], m["key_scale"], m["value_scale"],
        m["block_tables"], m["seq_lens"], None, 0.125, 1.0, 0)
    assert out.shape == m["query"].shape and out.dtype == F16 and out.device.type == "meta"
