"""What attention over a window and over a shared prefix refuse, checked without a GPU: the
Python entry points' ValueErrors, the C ABI's status codes, the traced ops' registration."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd import _lib, _op, build, shared_prefix, windowed  # noqa: E402,F401
from small_q_attention_amd.masks import spec_dec_mask  # noqa: E402

F16, BF16, E4M3, INT8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn, torch.int8


def _zeros(*shape, dtype=torch.float32):
    x = torch.zeros(*shape, dtype=torch.uint8 if dtype is E4M3 else dtype)
    return x.view(E4M3) if dtype is E4M3 else x


def _base(kv=F16, dtype=F16, b=3, q=3, hq=8, hkv=2, d=64, pages=6, page=16, width=4, scaled=False):
    return dict(query=_zeros(b, q, hq, d, dtype=dtype),
                key_cache=_zeros(pages, page, hkv, d, dtype=kv),
                value_cache=_zeros(pages, page, hkv, d, dtype=kv),
                block_tables=torch.zeros(b, width, dtype=torch.int32),
                seq_lens=torch.ones(b, dtype=torch.int32),
                key_scale=torch.ones(pages, hkv) if scaled else None,
                value_scale=torch.ones(pages, hkv) if scaled else None)


def _plan(groups=((0, 2, 2),), shape=(3, 3, 8, 2, 64, 16), device="cuda:0"):
    """A plan as the planner makes it, without a device to ask."""
    return shared_prefix.SharedPrefixPlan(tuple(shape), tuple(groups), torch.device(device),
                                          torch.zeros(1, dtype=torch.int32))


def _window(a, window=8, **kw):
    return windowed.paged_attention_windowed(window=window, **{**a, **kw})


def _prefix(a, plan=None, **kw):
    return shared_prefix.paged_attention_shared_prefix(plan=plan or _plan(), **{**a, **kw})


CALLS = {"window": _window, "prefix": _prefix}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change,match", [
    (dict(query=torch.zeros(3, 3, 8, dtype=F16)), "query must be"),
    (dict(query=torch.zeros(3, 3, 8, 64)), "float16 or bfloat16"),
    (dict(query=torch.zeros(3, 3, 9, 64, dtype=F16)), "multiple of its kv heads"),
    (dict(query=torch.zeros(3, 3, 8, 128, dtype=F16)), "head_dim"),
    (dict(query=torch.zeros(3, 17, 8, 64, dtype=F16)), "at most 64"),
    (dict(query=torch.zeros(3, 8, 3, 64, dtype=F16).transpose(1, 2)), "query must be"),
    (dict(key_cache=torch.zeros(6, 16, 2, 64, dtype=BF16),
          value_cache=torch.zeros(6, 16, 2, 64, dtype=BF16)), "query's type"),
    (dict(key_cache=torch.zeros(6, 16, 2, 64, dtype=INT8),
          value_cache=torch.zeros(6, 16, 2, 64, dtype=INT8)), "need key_scale"),
    (dict(value_cache=torch.zeros(6, 16, 2, 64, dtype=BF16)), "match"),
    (dict(key_cache=torch.zeros(6, 17, 2, 64, dtype=F16)), "page_size"),
    (dict(key_cache=torch.zeros(0, 16, 2, 64, dtype=F16)), "not empty"),
    (dict(key_scale=torch.ones(6, 2)), "come together"),
    (dict(key_scale=torch.ones(6, 2), value_scale=torch.ones(6, 2)), "scales belong"),
    (dict(block_tables=torch.zeros(3, 4)), "int32"),
    (dict(block_tables=torch.zeros(2, 4, dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros(3, 0, dtype=torch.int32)), "block_tables"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int32)), "seq_lens"),
    (dict(seq_lens=torch.ones(6, dtype=torch.int32)[::2]), "seq_lens"),
    (dict(scale=0.0), "scale must be"),
    (dict(scale=float("nan")), "scale must be"),
    (dict(scale=float("inf")), "scale must be"),
    (dict(mask=torch.zeros(3, 3, dtype=torch.int64)), "16- or 32-bit"),
    (dict(mask=torch.zeros(2, 3, 1, dtype=torch.int32)), "draft mask"),
    (dict(), "GPU tensor"),
])
def test_calls_refuse(call, change, match):
    with pytest.raises(ValueError, match=match):
        CALLS[call](_base(), **change)


@pytest.mark.parametrize("call", CALLS)
def test_scales_are_checked(call):
    for change, match in ((dict(value_scale=None), "come together"),
                          (dict(key_scale=torch.ones(6, 3)), "key_scale must be float32"),
                          (dict(value_scale=torch.ones(6, 2).half()), "value_scale must be"),
                          (dict(value_scale=torch.ones(6, 4)[:, ::2]), "must match")):
        with pytest.raises(ValueError, match=match):
            CALLS[call](_base(kv=INT8, scaled=True), **change)


@pytest.mark.parametrize("window,sink", [(0, 0), (-1, 0), (5, -1)])
def test_windows_are_checked(window, sink):
    with pytest.raises(ValueError, match="window must be positive"):
        _window(_base(), window=window, sink=sink)


def test_rows_at_head_dim_256():
    with pytest.raises(ValueError, match="at most 32 at head_dim 256"):
        _window(_base(d=256, q=9))


@pytest.mark.parametrize("groups,match", [
    ([(0, 2)], "groups are"), ([(-1, 2, 1)], "groups are"), ([(0, 0, 1)], "groups are"),
    ([(0, 4, 1)], "groups are"), ([(0, 2, -1)], "groups are"), ([(0, 2, 1), (1, 2, 1)], "groups are"),
    ([(1, 2, 1), (0, 1, 1)], "groups are"), ([(0, 2, 2**26)], "2\\^30"),
])
def test_plans_refuse_groups(groups, match):
    with pytest.raises(ValueError, match=match):
        shared_prefix.plan_shared_prefix(groups, 3, 3, 8, 2, 64, 16)


@pytest.mark.parametrize("change,match", [
    (dict(batch=0), "positive"), (dict(q_len=0), "positive"), (dict(num_query_heads=9), "multiple"),
    (dict(head_dim=96), "head_dim"), (dict(page_size=48), "page_size"), (dict(q_len=17), "at most"),
    (dict(head_dim=256, q_len=9), "at most 32"), (dict(device="cpu"), "must be a GPU"),
])
def test_plans_refuse_shapes(change, match):
    shape = dict(batch=3, q_len=3, num_query_heads=8, num_kv_heads=2, head_dim=64, page_size=16)
    with pytest.raises(ValueError, match=match):
        shared_prefix.plan_shared_prefix([(0, 2, 1)], **{**shape, **change})


def test_a_plan_serves_its_shape_only():
    with pytest.raises(ValueError, match="plan_shared_prefix"):
        _prefix(_base(), plan="a plan")
    # (Host tensors are refused before a plan's shape is looked at.)
    a = _base()
    for change, match in ((dict(shape=(3, 2, 8, 2, 64, 16)), "made for"),
                          (dict(groups=((0, 2, 5),)), "shares 5 pages")):
        with pytest.raises(ValueError, match=match):
            _check_on_device(a, _plan(device="cpu", **change))


def _check_on_device(a, plan):
    """The plan's checks, as if the tensors lived where the plan does."""
    import unittest.mock as mock

    with mock.patch.object(shared_prefix, "check_call"):
        shared_prefix._check(a["query"], a["key_cache"], a["value_cache"], None, None,
                             a["block_tables"], a["seq_lens"], None, plan, None, None)


def test_out_is_not_the_query():
    q = torch.zeros(2, 3, dtype=F16)
    windowed.check_apart(q, None)
    windowed.check_apart(q, torch.zeros(2, 3, dtype=F16))
    with pytest.raises(ValueError, match="must not be query"):
        windowed.check_apart(q, q.view(2, 3))


# --------------------------------------------------------------------------------------
# The C ABI.
# --------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def lib():
    if build.is_stale():
        build.build()
    return _lib.load()


def _args(**kw):
    buf = 1 << 20  # never followed: every call here is refused
    base = dict(struct_size=ctypes.sizeof(_lib.AttentionArgs), query=buf, output=buf,
                block_tables=buf, seq_lens=buf, max_pages=4, scale=0.1, out_scale=1.0, batch=3,
                q_len=3, num_query_heads=8, num_kv_heads=2, head_dim=64, page_size=16, num_splits=2,
                pages_per_split=1, workspace=buf, workspace_bytes=1 << 30, dtype=_lib.DTYPE_F16,
                kv_dtype=_lib.DTYPE_F16)
    kv = dict(k=buf, v=buf, num_pages=6, page_stride=2048, token_stride=128, head_stride=64)
    kv.update({k[3:]: v for k, v in kw.items() if k.startswith("kv_") and k != "kv_dtype"})
    base.update({k: v for k, v in kw.items() if not k.startswith("kv_") or k == "kv_dtype"})
    a = _lib.AttentionArgs(**base)
    a.kv = _lib.KVCache(**kv)
    return a


def _c_plan(**kw):
    base = dict(struct_size=ctypes.sizeof(_lib.SharedPlan), batch=3, q_len=3, num_query_heads=8,
                num_kv_heads=2, head_dim=64, page_size=16, num_groups=1, most_pages=2, num_splits=2,
                pages_per_split=1, wg_heads=2, block_rows=32, shared_size=2, shared_splits=1,
                num_items=1)
    base.update(kw)
    return _lib.SharedPlan(**base)


BAD = [
    (dict(struct_size=8), 1, "struct_size"), (dict(query=0), 1, "null"),
    (dict(kv_k=0), 1, "null"), (dict(batch=0), 1, "positive"), (dict(q_len=-1), 1, "positive"),
    (dict(num_query_heads=9), 1, "divisible"), (dict(head_dim=96), 2, "head_dim"),
    (dict(q_len=17), 2, "exceeds 64"), (dict(page_size=24), 2, "page_size"),
    (dict(kv_num_pages=0), 1, "empty"), (dict(kv_num_pages=2**31), 1, "32 bits"),
    (dict(max_pages=0), 1, "empty"), (dict(max_pages=2**26), 1, "2^30"),
    (dict(dtype=_lib.DTYPE_INT8), 2, "dtype"), (dict(kv_dtype=_lib.DTYPE_BF16), 2, "kv_dtype"),
    (dict(kv_dtype=_lib.DTYPE_INT8), 1, "need scales"), (dict(kv_token_stride=4), 1, "multiples"),
    (dict(kv_page_stride=-8), 1, "non-negative"), (dict(kv_k=24), 1, "aligned"),
    (dict(kv_page_stride=2**41), 1, "too large"), (dict(kv_token_stride=2**30 - 8), 1, "2 GiB"),
    (dict(query=8 + (1 << 20)), 1, "aligned"), (dict(seq_lens=2 + (1 << 20)), 1, "aligned"),
    (dict(draft_mask=1 << 20, mask_words=0), 1, "draft_mask"),
    (dict(draft_mask=1 << 20, mask_words=3), 1, "draft_mask"), (dict(scale=0.0), 1, "scale"),
    (dict(out_scale=float("inf")), 1, "finite"), (dict(flags=1), 1, "flags"),
    (dict(pages_per_split=2), 1, "pages_per_split"), (dict(num_splits=0), 1, "num_splits"),
    (dict(pages_per_split=0, num_splits=3), 1, "num_splits"),
    (dict(workspace=0), 3, "workspace"), (dict(workspace_bytes=16), 3, "workspace"),
    (dict(workspace=8 + (1 << 20)), 3, "aligned"),
    (dict(num_splits=2**28), 1, "grid too large"),
]


@pytest.mark.parametrize("change,status,match", BAD)
def test_windowed_status(lib, change, status, match):
    assert lib.sqa_paged_attention_windowed(ctypes.byref(_args(**change)), None, 10, 0, 2) == status
    assert match in lib.sqa_last_error().decode()


@pytest.mark.parametrize("change,status,match", [x for x in BAD if "num_splits" not in x[0]
                                                 and "pages_per_split" not in x[0]])
def test_shared_prefix_status(lib, change, status, match):
    rc = lib.sqa_paged_attention_shared_prefix(ctypes.byref(_args(**change)), None,
                                               ctypes.byref(_c_plan()), 1 << 20)
    # (A plan of another shape is found out before, where the change is one of shape.)
    text = lib.sqa_last_error().decode()
    assert rc == status and match in text or "another batch" in text


def test_window_arguments(lib):
    for window, sink, heads in ((0, 0, 2), (-5, 0, 2), (3, -1, 2), (3, 0, 3), (3, 0, 0), (3, 0, 8)):
        assert lib.sqa_paged_attention_windowed(ctypes.byref(_args()), None, window, sink, heads) == 1
    assert lib.sqa_paged_attention_windowed(None, None, 3, 0, 2) == 1
    scales = _lib.BlockScales(k=1 << 20, v=1 << 20, page_stride=2, head_stride=1)
    assert lib.sqa_paged_attention_windowed(ctypes.byref(_args()), ctypes.byref(scales), 3, 0, 2) == 1
    codes = _args(kv_dtype=_lib.DTYPE_INT8)
    for bad in (dict(k=0), dict(v=0), dict(k=2 + (1 << 20)), dict(page_stride=-1),
                dict(head_stride=2**30)):
        s = _lib.BlockScales(**{**dict(k=1 << 20, v=1 << 20, page_stride=2, head_stride=1), **bad})
        assert lib.sqa_paged_attention_windowed(ctypes.byref(codes), ctypes.byref(s), 3, 0, 2) == 1


@pytest.mark.parametrize("change", [
    dict(struct_size=4), dict(batch=2), dict(q_len=2), dict(num_query_heads=4), dict(page_size=32),
    dict(num_splits=3), dict(pages_per_split=0, num_splits=3), dict(most_pages=5),
    dict(block_rows=48), dict(block_rows=256, head_dim=64, num_items=-1), dict(shared_size=0),
    dict(shared_splits=-1), dict(num_groups=0), dict(block_rows=8), dict(wg_heads=3)])
def test_shared_prefix_refuses_plans(lib, change):
    rc = lib.sqa_paged_attention_shared_prefix(ctypes.byref(_args()), None,
                                               ctypes.byref(_c_plan(**change)), 1 << 20)
    assert rc == 1, lib.sqa_last_error()


def test_shared_prefix_needs_its_table(lib):
    for table in (0, 2 + (1 << 20)):
        assert lib.sqa_paged_attention_shared_prefix(ctypes.byref(_args()), None,
                                                     ctypes.byref(_c_plan()), table) == 1
    assert lib.sqa_paged_attention_shared_prefix(ctypes.byref(_args()), None, None, 1 << 20) == 1
    assert lib.sqa_shared_workspace_bytes(None) == 0
    assert lib.sqa_shared_workspace_bytes(ctypes.byref(_c_plan(struct_size=1))) == 0


def test_workspace_of_a_plan(lib):
    rows = 3 * 8  # a sequence's, all heads
    floats = 64 + 2
    assert lib.sqa_shared_workspace_bytes(ctypes.byref(_c_plan())) == (2 + 1) * 3 * rows * floats * 4
    assert lib.sqa_shared_workspace_bytes(ctypes.byref(_c_plan(num_items=0, num_splits=1,
                                                               shared_splits=0))) == 0
    crossing = _c_plan(pages_per_split=0, num_splits=11)
    assert lib.sqa_shared_workspace_bytes(ctypes.byref(crossing)) == \
        (11 + 3) * rows * floats * 4 + 3 * 8


def test_plans_without_a_device(lib):
    """Arguments are checked before the device is asked for."""
    n = ctypes.c_int()
    out = (ctypes.byref(n),) * 3
    for shape, window, sink, pages in (((0, 1, 8, 2, 64), 5, 0, 4), ((2, 1, 8, 3, 64), 5, 0, 4),
                                       ((2, 1, 8, 2, 65), 5, 0, 4), ((2, 1, 8, 2, 64), 0, 0, 4),
                                       ((2, 1, 8, 2, 64), 5, -1, 4), ((2, 1, 8, 2, 64), 5, 0, 0)):
        assert lib.sqa_plan_windowed(0, *shape, window, sink, 0, pages, 0, *out) in (1, 2)
    groups = (ctypes.c_int32 * 3)(0, 2, 5)
    plan = _lib.SharedPlan()
    good = [0, 3, 3, 8, 2, 64, 16, 0, 1, groups, 0, 4, ctypes.byref(plan), None]
    for i, bad in ((12, None), (1, 0), (6, 20), (8, -1), (9, None), (11, 0), (11, 2**26)):
        a = list(good)
        a[i] = bad
        assert lib.sqa_plan_shared_prefix(*a) in (1, 2), i


def test_traced_ops_are_registered():
    q, k = torch.empty(3, 3, 8, 64, dtype=F16, device="meta"), torch.empty(6, 16, 2, 64, dtype=F16,
                                                                           device="meta")
    t = torch.empty(3, 4, dtype=torch.int32, device="meta")
    n = torch.empty(3, dtype=torch.int32, device="meta")
    out = torch.ops.sqa.paged_attention_windowed(q, k, k, None, None, t, n, None, 8, 0, 0.1, 1.0, 0)
    assert out.shape == q.shape and out.dtype == F16
    out = torch.ops.sqa.paged_attention_shared_prefix(q, k, k, None, None, t, n, None, [0, 2, 1], n,
                                                      0.1, 1.0, 0)
    assert out.shape == q.shape
    assert spec_dec_mask(1, 2).shape == (1, 2, 2)


def test_a_plans_table_is_held_for_each_stream(monkeypatch):
    """Once for a stream of eager calls, every time where no plan counts them, never under
    capture."""
    held, capturing = [], [False]

    class Table:
        def record_stream(self, stream):
            held.append(stream)

    monkeypatch.setattr(_lib, "_CUDA_STATE", (lambda: 0, lambda: capturing[0]))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: f"current of {device}")
    seen = _plan().streams
    for stream, streams, count in ((7, seen, 1), (7, seen, 1), (9, seen, 2), (9, None, 3),
                                   (9, None, 4)):
        shared_prefix.hold_table(Table(), stream, "cuda:0", streams)
        assert len(held) == count
    capturing[0] = True
    shared_prefix.hold_table(Table(), 11, "cuda:0", seen)
    assert len(held) == 4 and seen == {7, 9} and held[0] == "current of cuda:0"


def test_out_does_not_overlap_the_query():
    """A result that begins within the queries, or they within it, is refused; one that begins
    where they end is not."""
    store = torch.zeros(40, dtype=F16)
    q = store[8:24].view(2, 8)
    for at in (0, 1, 7, 9, 16, 23):
        with pytest.raises(ValueError, match="overlap"):
            windowed.check_apart(q, store[at:at + 16].view(2, 8))
    windowed.check_apart(store[:16].view(2, 8), store[16:32].view(2, 8))
    windowed.check_apart(store[16:32].view(2, 8), store[:16].view(2, 8))


@pytest.mark.parametrize("off", [0, 16, -16, 3 * 3 * 8 * 64 * 2 - 8, -(3 * 3 * 8 * 64 * 2 - 8)])
def test_c_entries_refuse_an_output_over_the_query(lib, off):
    a = _args(output=(1 << 20) + off)
    assert lib.sqa_paged_attention_windowed(ctypes.byref(a), None, 10, 0, 2) == 1
    assert "overlaps" in lib.sqa_last_error().decode()
    assert lib.sqa_paged_attention_shared_prefix(ctypes.byref(a), None, ctypes.byref(_c_plan()),
                                                 1 << 20) == 1
    assert "overlaps" in lib.sqa_last_error().decode()


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("factors", [
    dict(out_scale=float("nan")), dict(out_scale=float("inf")), dict(out_scale=-float("inf")),
    dict(out_scale=2.0 ** 128), dict(scale=2.0 ** 128), dict(scale=1e300), dict(scale=2.0 ** -150)])
def test_factors_that_32_bits_do_not_hold(call, factors):
    with pytest.raises(ValueError, match="in 32 bits"):
        CALLS[call](_base(), **factors)
    assert windowed.check_factors(None, -2.0, 64) == (0.125, -2.0)
    assert windowed.check_factors(2.0 ** -149, 3.4028234e38, 64) == (2.0 ** -149, 3.4028234e38)


def test_what_the_library_refuses_is_a_value_error(lib):
    """Alignments, strides and workspaces that only the C entries look at."""
    a = _base()
    store = torch.zeros(a["query"].numel() + 8, dtype=F16)
    args = lambda **kw: [{**a, "out": store[:-8].view(a["query"].shape), **kw}[n] for n in (  # noqa: E731
        "query", "out", "key_cache", "value_cache", "key_scale", "value_scale", "block_tables",
        "seq_lens")]
    odd = store[1:a["query"].numel() + 1].view(a["query"].shape)
    # (Never touched, so never more than addresses.)
    far = torch.empty(15 << 27 | 128, dtype=F16).as_strided((6, 16, 2, 64), (0, 1 << 27, 64, 1))
    ws = torch.zeros(1 << 20, dtype=torch.uint8)[4:]
    plan = _c_plan()
    for launch, rest in ((_lib.launch_windowed, (None, 8, 0, 0.1, 1.0, (2, 1, 2))),
                         (_lib.launch_shared_prefix, (None, plan, torch.zeros(32, dtype=torch.int32),
                                                      0.1, 1.0))):
        for change, space, match in ((dict(out=odd), None, "aligned"),
                                     (dict(key_cache=far, value_cache=far), None, "2 GiB"),
                                     ({}, ws, "aligned"), ({}, ws[:16], "workspace of")):
            with pytest.raises(ValueError, match=match):
                launch(*args(**change), *rest, space, 0)
    with pytest.raises(ValueError, match="grid too large"):
        _lib.plan_windowed(0, 2**20, 16, 2**10, 2**10, 64, 5, 0, 0, 4, 0)
    assert isinstance(_lib.refusal(lib, "x", _lib.SQA_ERR_HIP), RuntimeError)


@pytest.mark.parametrize("change,status,match", [x for x in BAD if "num_splits" not in x[0]
                                                 and "pages_per_split" not in x[0]])
def test_shared_prefix_names_what_it_refuses(lib, change, status, match):
    """Each by its own check, not by the plan's other shape."""
    rc = lib.sqa_paged_attention_shared_prefix(ctypes.byref(_args(**change)), None,
                                               ctypes.byref(_c_plan()), 1 << 20)
    assert rc == status
    assert match in lib.sqa_last_error().decode()


@pytest.mark.parametrize("shape", [dict(batch=2), dict(q_len=2), dict(num_query_heads=4),
                                   dict(num_kv_heads=1), dict(head_dim=128), dict(page_size=32),
                                   dict(num_splits=3), dict(num_splits=9, pages_per_split=0)])
def test_shared_prefix_refuses_a_plan_of_another_shape(lib, shape):
    strides = dict(kv_page_stride=2**16, kv_token_stride=512)
    for a, plan in ((_args(**strides), _c_plan(**shape)), (_args(**strides, **shape), _c_plan())):
        assert lib.sqa_paged_attention_shared_prefix(ctypes.byref(a), None, ctypes.byref(plan),
                                                     1 << 20) == 1
        assert "another batch" in lib.sqa_last_error().decode()


@pytest.mark.parametrize("shape,plan", [
    ({}, dict(block_rows=48)), ({}, dict(block_rows=8)), ({}, dict(block_rows=0)),
    ({}, dict(block_rows=512)), (dict(q_len=12), dict(block_rows=32)),
    (dict(q_len=12), dict(block_rows=256)), (dict(head_dim=256), dict(block_rows=64)),
    (dict(head_dim=256), dict(block_rows=256)), ({}, dict(shared_splits=0))])
def test_shared_prefix_refuses_blocks_that_no_kernel_has(lib, shape, plan):
    """Plans that agree with the call in all but how the groups are cut."""
    a = _args(**shape, kv_page_stride=2**16, kv_token_stride=512)
    assert lib.sqa_paged_attention_shared_prefix(ctypes.byref(a), None,
                                                 ctypes.byref(_c_plan(**shape, **plan)),
                                                 1 << 20) == 1
    assert lib.sqa_last_error().decode() == "not a plan of sqa_plan_shared_prefix"


def test_calls_are_planned_by_pages():
    """Lengths on one page are one to the plans and their caches."""
    for n, pages in ((-3, 0), (0, 0), (1, 16), (16, 16), (17, 32), (8191, 8192),
                     (2**31 - 1, 2**31 - 16), (2**40, 2**31 - 16)):
        assert windowed.whole_pages(n) == pages
