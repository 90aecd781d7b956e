"""Attention over a window and the first tokens on the GPU, against a plain statement in
64 bits."""

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd.masks import pack_draft_mask  # noqa: E402
from small_q_attention_amd.windowed import paged_attention_windowed  # noqa: E402
from tests import _part_reference as ref  # noqa: E402
from tests._part_reference import BF16, E4M3, F16, INT8  # noqa: E402

pytestmark = pytest.mark.gpu

CACHES = [(F16, None, False), (BF16, None, False), (F16, E4M3, False), (BF16, E4M3, False),
          (F16, E4M3, True), (BF16, INT8, True)]


def _check(lens, q_len, hq, hkv, d, page, dtype, kv, scaled, window, sink, seed=0, tree=None,
           splits=True, **kw):
    q, caches, scales, tables, sl = ref.window_inputs(lens, q_len, hq, hkv, d, page, dtype, kv,
                                                      scaled, window, sink, seed, **kw)
    want, bound = ref.attention(
        q, *caches, *scales, tables, sl,
        lambda i, n: ref.window_seen(n, q_len, window, sink, None if tree is None else tree[i]))
    qc, kc, vc, ks, vs, bt, slc = ref.cuda(q, *caches, *scales, tables, sl)
    mask = None if tree is None else pack_draft_mask(tree).cuda()
    outs = []
    for most in (0, max(max(lens), 1)):
        out = paged_attention_windowed(qc, kc, vc, bt, slc, window, sink=sink, key_scale=ks,
                                       value_scale=vs, max_seq_len=most, mask=mask)
        ref.assert_within(out, want, bound, f"max_seq_len {most}")
        outs.append(out)
    again = paged_attention_windowed(qc, kc, vc, bt, slc, window, sink=sink, key_scale=ks,
                                     value_scale=vs, mask=mask)
    assert torch.equal(outs[0], again)


LENS = [777, 0, 1, 15, 16, 17, 40, 300, 5]


@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
@pytest.mark.parametrize("window,sink", [(1, 0), (2, 1), (15, 4), (16, 16), (17, 0), (33, 17),
                                         (100, 40), (290, 500), (2000, 3)])
def test_windows_and_first_tokens(dtype, kv, scaled, window, sink):
    _check(LENS, 3, 8, 2, 128, 16, dtype, kv, scaled, window, sink, seed=window)


@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
@pytest.mark.parametrize("q_len,hq,hkv,d,page", [
    (1, 8, 8, 128, 16), (1, 32, 8, 128, 32), (16, 16, 4, 128, 64), (7, 15, 3, 128, 256),
    (5, 5, 5, 64, 16), (1, 8, 1, 64, 64), (8, 32, 4, 64, 32), (2, 16, 2, 256, 16),
    (8, 8, 2, 256, 128), (16, 4, 4, 64, 16)])
def test_shapes(dtype, kv, scaled, q_len, hq, hkv, d, page):
    _check([500, 33, 1200, 260], q_len, hq, hkv, d, page, dtype, kv, scaled, 150, 20, seed=q_len)


@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
@pytest.mark.parametrize("window", [1, 3, 60])
def test_draft_trees_and_rows_that_see_nothing(dtype, kv, scaled, window):
    """Trees whose rows 0 and 2 see no draft token: with a window of one and no first tokens
    those rows see nothing at all and are 0."""
    lens = [100, 4, 6, 250]
    tree = ref.trees(len(lens), 4, seed=3, empty=(0, 2))
    _check(lens, 4, 8, 2, 128, 16, dtype, kv, scaled, window, 0, seed=5, tree=tree)
    _check(lens, 4, 8, 2, 128, 16, dtype, kv, scaled, window, 9, seed=5, tree=tree)


@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
def test_long_streams_in_many_splits(dtype, kv, scaled):
    _check([9000, 8191, 4097], 4, 8, 2, 128, 16, dtype, kv, scaled, 4096, 64, seed=8)
    _check([20011], 1, 4, 1, 128, 64, dtype, kv, scaled, 8192, 5, seed=9)


@pytest.mark.parametrize("b", [1, 63, 65, 130, 300])
def test_batches(b):
    lens = [(37 * i) % 191 + 1 for i in range(b)]
    _check(lens, 2, 4, 2, 64, 16, F16, None, False, 50, 7, seed=b)


@pytest.mark.parametrize("kv", [E4M3, INT8])
def test_blocks_of_unlike_scales(kv):
    _check([700, 90], 4, 8, 2, 128, 16, F16, kv, True, 300, 30, seed=4, quiet=False)


@pytest.mark.parametrize("dtype,kv", [(F16, None), (BF16, None), (F16, E4M3)])
@pytest.mark.parametrize("q_len", [3, 8, 16])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(dtype, kv, q_len):
    """NaN (and infinities where the type has them) at the window's edge, in a first token
    and in the draft block."""
    hkv, d, page, window, sink = 2, 128, 16, 40, 5
    lens = [200, 120]
    q, caches, scales, tables, sl = ref.window_inputs(lens, q_len, 4 * hkv, hkv, d, page, dtype, kv,
                                                      False, window, sink, seed=q_len)

    def put(c, i, t, h, e, x):
        raw = c.view(torch.uint8) if c.element_size() == 1 else c
        raw[int(tables[i, t // page]), t % page, h, e] = 0x7F if c.element_size() == 1 else x

    k, v = caches
    nan, inf = float("nan"), float("inf")
    put(v, 0, 199 - window, 1, 7, nan)            # seen by all rows but the last
    put(v, 0, 200 - q_len + 1 - window, 0, 3, inf)  # by row 0 alone
    put(v, 0, 2, 0, 70, -inf)                     # a first token: by all
    put(v, 0, 200 - q_len + 1, 1, 9, -inf)        # draft token 1
    put(v, 0, 199, 1, 9, inf)                     # the last draft token
    put(k, 1, 120 - q_len + 1, 0, 5, nan)
    put(k, 1, 119 - window, 1, 5, nan)
    seen = lambda i, n: ref.window_seen(n, q_len, window, sink)  # noqa: E731
    want, bound = ref.attention(q, k, v, None, None, tables, sl, seen)
    assert want.isnan().any() and want.isfinite().any()
    qc, kc, vc, bt, slc = ref.cuda(q, k, v, tables, sl)
    out = paged_attention_windowed(qc, kc, vc, bt, slc, window, sink=sink)
    ref.assert_within(out, want, bound)


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("kv", [None, E4M3])
def test_interleaved_caches(layout, kv):
    lens, q_len, hkv, d, page = [300, 77], 4, 4, 128, 32
    q, (k, v), _, tables, sl = ref.window_inputs(lens, q_len, 16, hkv, d, page, F16, kv, False, 64,
                                                 10)
    want, bound = ref.attention(q, k, v, None, None, tables, sl,
                                lambda i, n: ref.window_seen(n, q_len, 64, 10))
    raw = [c.view(torch.uint8) if kv else c for c in (k, v)]
    if layout == "HND":
        raw = [c.transpose(1, 2) for c in raw]
    both = torch.stack(raw, 1).contiguous().cuda()
    both = both.view(kv) if kv else both
    views = [both[:, 0], both[:, 1]]
    if layout == "HND":
        views = [c.transpose(1, 2) for c in views]
    qc, bt, slc = ref.cuda(q, tables, sl)
    out = paged_attention_windowed(qc, *views, bt, slc, 64, sink=10)
    ref.assert_within(out, want, bound)


def test_a_window_over_everything_is_attention_over_everything():
    from small_q_attention_amd.cuda import paged_mtp_attention

    q, (k, v), _, tables, sl = ref.window_inputs([1000, 333], 4, 32, 8, 128, 16, F16, None, False,
                                                 1 << 20, 0)
    tables = tables.clamp(min=0)
    qc, kc, vc, bt, slc = ref.cuda(q, k, v, tables, sl)
    a = paged_attention_windowed(qc, kc, vc, bt, slc, 2**31 - 1)
    b = paged_mtp_attention(qc, kc, vc, bt, slc)
    assert (a.float() - b.float()).abs().max() <= 2e-3


def test_scales_out_and_workspace():
    q, (k, v), _, tables, sl = ref.window_inputs([3000, 901], 4, 8, 2, 128, 16, F16, None, False,
                                                 700, 3)
    want, bound = ref.attention(q, k, v, None, None, tables, sl,
                                lambda i, n: ref.window_seen(n, 4, 700, 3), scale=0.05,
                                out_scale=-1.5)
    qc, kc, vc, bt, slc = ref.cuda(q, k, v, tables, sl)
    out = torch.empty_like(qc)
    ws = torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")
    got = paged_attention_windowed(qc, kc, vc, bt, slc, 700, sink=3, scale=0.05, out_scale=-1.5,
                                   out=out, workspace_buffer=ws)
    assert got is out
    ref.assert_within(out, want, bound)
    with pytest.raises(ValueError, match="workspace_buffer"):
        paged_attention_windowed(qc, kc, vc, bt, slc, 700, sink=3, workspace_buffer=ws[:64])


def test_lengths_past_the_table_and_ids_outside_the_pool():
    """A length past the table row is held to its pages; ids outside the pool stand for page
    0. Neither reads out of bounds."""
    q, (k, v), _, tables, sl = ref.window_inputs([64, 64], 2, 4, 2, 64, 16, F16, None, False, 30, 0)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    qc, kc, vc, bt, _ = ref.cuda(q, k, v, tables, sl)
    for n in (65, 10**6, 2**31 - 1, -5):
        lens = torch.tensor([n, 64], dtype=torch.int32, device="cuda")
        out = paged_attention_windowed(qc, kc, vc, bt, lens, 30)
        assert torch.isfinite(out).all()
        assert n > 0 or not out[0].any()
    bad = bt.clone()
    bad[0] = 10**6
    lens = torch.tensor([64, 64], dtype=torch.int32, device="cuda")
    zero = bt.clone()
    zero[0] = 0
    assert torch.equal(paged_attention_windowed(qc, kc, vc, bad, lens, 30),
                       paged_attention_windowed(qc, kc, vc, zero, lens, 30))
