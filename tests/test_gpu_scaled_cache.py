"""8-bit caches with block scales on the GPU: the quantising append and attention, against
plain statements in 64 bits."""

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd.masks import pack_draft_mask  # noqa: E402
from small_q_attention_amd.scaled_cache import (append_scaled_kv,  # noqa: E402
                                                paged_attention_scaled)
from tests import _cache_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3, INT8, F16, BF16 = torch.float8_e4m3fn, torch.int8, torch.float16, torch.bfloat16
NAN_CODE = 0x7F


def _tables(lens, page, pool, gen, width=None, pad=-1):
    used = [-(-max(n, 0) // page) for n in lens]
    perm = torch.randperm(pool, generator=gen).to(torch.int32)
    tables = torch.full((len(lens), width or max(max(used), 1)), pad, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        tables[i, :n] = perm[at:at + n]
        at += n
    return tables, perm[at:]


def _inputs(lens, q_len, hq, hkv, d, page, dtype, kv, seed=0, width=None, quiet=False):
    """Query, codes, scales, tables, lengths on the CPU. Blocks differ in size by up to
    2^12; slots past a sequence's end and pages nobody owns hold NaN codes (or the lowest
    integer) and NaN scales."""
    g = torch.Generator().manual_seed(seed)
    pool = sum(-(-max(n, 0) // page) for n in lens) + 3
    tables, free = _tables(lens, page, pool, g, width)
    q = torch.randn(len(lens), q_len, hq, d, generator=g).to(dtype)
    caches, scales = [], []
    for which in range(2):
        x = torch.randn(pool, page, hkv, d, generator=g)
        size = 2.0 ** torch.randint(-8 if which else -3, 5 if which else 2, (pool, 1, hkv, 1),
                                    generator=g)
        codes, scale = ref.quantise(x * size, kv)
        raw = codes.view(torch.uint8)
        junk = NAN_CODE if kv is E4M3 else 0x80
        raw[free.long()] = junk
        scale[free.long()] = float("nan")
        for i, n in enumerate(lens):
            if n > 0 and n % page:
                raw[int(tables[i, n // page]), n % page:] = junk
        caches.append(codes)
        scales.append(scale)
    return q, caches, scales, tables, torch.tensor(lens, dtype=torch.int32)


def _trees(b, q_len, seed=0, empty=()):
    """Random draft trees; rows in ``empty`` see no draft token."""
    g = torch.Generator().manual_seed(seed)
    seen = torch.rand(b, q_len, q_len, generator=g) < 0.5
    for r in empty:
        if r < q_len:
            seen[:, r] = False
    return seen


def _cuda(*xs):
    return [x.cuda() for x in xs]


def _check(lens, q_len, hq, hkv, d, page, dtype, kv, seed=0, trees=None, **kw):
    q, caches, scales, tables, sl = _inputs(lens, q_len, hq, hkv, d, page, dtype, kv, seed,
                                            kw.pop("width", None))
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl, trees)
    qc, kc, vc, ks, vs, bt, slc = _cuda(q, *caches, *scales, tables, sl)
    mask = None if trees is None else pack_draft_mask(trees).cuda()
    for most in (0, max(max(lens), 1)):
        out = paged_attention_scaled(qc, kc, vc, ks, vs, bt, slc, max_seq_len=most, mask=mask)
        ref.assert_within(out, want, bound, f"max_seq_len {most}")
    again = paged_attention_scaled(qc, kc, vc, ks, vs, bt, slc, mask=mask)
    assert torch.equal(out, again)  # the length given only sizes the call; same bits


@pytest.mark.parametrize("kv", [E4M3, INT8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("q_len,group", [(1, 1), (1, 4), (4, 4), (5, 3), (8, 4), (9, 7), (16, 4)])
def test_attention_rows(q_len, group, dtype, kv):
    _check([777, 41, 2048, q_len], q_len, 4 * group, 4, 128, 16, dtype, kv, seed=q_len)


@pytest.mark.parametrize("kv", [E4M3, INT8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("d,q_len", [(64, 2), (64, 7), (64, 16), (256, 3), (256, 8)])
def test_attention_head_dims(d, q_len, kv):
    _check([1500, 17, 333], q_len, 16, 4, d, 32, F16, kv, seed=d)
    _check([1500, 17, 333], q_len, 16, 4, d, 32, BF16, kv, seed=d + 1)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("hkv", [1, 2, 3, 5, 8])
def test_attention_pages_and_heads(page, hkv):
    _check([1111, 256, 255, 1], 2, 4 * hkv, hkv, 128, page, F16, E4M3, seed=page + hkv)


@pytest.mark.parametrize("lens", [
    [0], [1], [2], [3], [15, 16, 17], [0, 0, 0], [64, 65, 0, 1], [5000], [1, 4097, 0, 300],
    [3] * 70, [33 * (i % 9) for i in range(300)], [16385, 1, 2]])
def test_attention_lengths(lens):
    """Empty sequences, rows that see nothing (fewer tokens than rows), one long sequence
    among short ones, more sequences than a wave has lanes or the chip work items."""
    _check(lens, 3, 8, 2, 64, 16, F16, E4M3, seed=len(lens), width=max(max(lens) // 16 + 2, 3))


@pytest.mark.parametrize("b", [65, 100, 127, 128, 129, 200])
def test_attention_batches_about_as_large_as_the_chip(b):
    """Lengths that differ, one of them far longer, in batches with few work items to spare
    and with none (eight kv heads: 128 items)."""
    lens = [(37 * i * i) % 700 for i in range(b)]
    lens[b // 3] = 9000
    q, caches, scales, tables, sl = _inputs(lens, 2, 8, 8, 64, 16, F16, INT8, b)
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl)
    args = _cuda(q, *caches, *scales, tables, sl)
    for most in (0, 9000, 1):  # the length only sizes the call
        ref.assert_within(paged_attention_scaled(*args, max_seq_len=most), want, bound, most)


@pytest.mark.parametrize("kv", [E4M3, INT8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("q_len", [1, 6, 16])
def test_attention_draft_trees(q_len, kv):
    lens = [600, q_len, 33 + q_len, q_len + 1]
    _check(lens, q_len, 8, 2, 128, 16, F16, kv, seed=q_len, trees=_trees(4, q_len, 1, (0, 3)))


def test_attention_nan_stays_with_the_rows_that_see_it():
    """NaN codes of draft tokens, K and V, reach the rows that see the token and no other;
    so does the scale of a page of the draft block."""
    q, caches, scales, tables, sl = _inputs([50], 8, 8, 2, 128, 16, F16, E4M3, seed=3)
    last = int(tables[0, 3])           # tokens 48 and 49: draft tokens 6 and 7
    caches[1].view(torch.uint8)[last, 0, 0, 5] = NAN_CODE   # V of token 48, head 0, dim 5
    caches[0].view(torch.uint8)[last, 1, 1, 9] = NAN_CODE   # K of token 49, head 1
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl)
    assert torch.isnan(want[0, 6:, :4, 5]).all() and torch.isnan(want[0, 7, 4:]).all()
    assert torch.isnan(want).sum() == 2 * 4 + 4 * 128
    out = paged_attention_scaled(*_cuda(q, *caches, *scales, tables, sl))
    ref.assert_within(out, want, bound)
    for which in range(2):
        scales2 = [s.clone() for s in scales]
        scales2[which][last, 1] = float("nan")
        out = paged_attention_scaled(*_cuda(q, *caches, *scales2, tables, sl))
        assert torch.isnan(out[0, 6:, 4:]).all() and not torch.isnan(out[0, :6]).any()


def test_attention_blocks_of_zeros():
    """Scale 0: the block's keys score 0, its values add nothing."""
    q, caches, scales, tables, sl = _inputs([200, 31], 4, 8, 2, 128, 16, F16, INT8, seed=4)
    for s in scales:
        s[tables[0, 2].long()] = 0.0
        s[tables[0, 12].long()] = 0.0  # the page of the draft block
        s[tables[1, :2].long()] = 0.0
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl)
    out = paged_attention_scaled(*_cuda(q, *caches, *scales, tables, sl))
    ref.assert_within(out, want, bound)
    assert (out[1] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("loud", [-30, -12, 8])
def test_attention_blocks_of_zeros_beside_others(loud, dtype):
    """Blocks of zeros that attract most of the attention, beside blocks of any size: what
    those hold is still there in the result."""
    q, caches, scales, tables, sl = _inputs([400, 90], 3, 8, 2, 128, 16, dtype, E4M3, seed=14)
    scales[1][tables[0, ::2].long()] = 0.0
    scales[0][tables[0, ::2].long()] *= 4.0
    scales[1][tables[0, 1::2].long()] *= 2.0 ** loud
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl)
    # The output's 2^-24 is for fp16's subnormals; bf16 has the range.
    if dtype is BF16:
        bound = bound - 2.0 ** -24 + 2.0 ** -60
    out = paged_attention_scaled(*_cuda(q, *caches, *scales, tables, sl))
    ref.assert_within(out, want, bound)
    assert dtype is F16 or (out[0].abs() > 0).float().mean() > 0.99


def test_attention_v_scales_far_apart():
    """Blocks of zeros beside blocks of scales up to 2^29, within the 2^100 that the scales may
    lie apart: what the blocks of zeros weigh is not lost."""
    q, caches, scales, tables, sl = _inputs([400, 90], 3, 8, 2, 128, 16, BF16, E4M3, seed=15)
    scales[1][tables[0, ::2].long()] = 0.0
    scales[0][tables[0, ::2].long()] *= 4.0
    scales[1][tables[0, 1::2].long()] *= 2.0 ** 32
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl)
    out = paged_attention_scaled(*_cuda(q, *caches, *scales, tables, sl))
    ref.assert_within(out, want, bound)


@pytest.mark.parametrize("layout", ["nhd", "hnd", "scales_together"])
def test_attention_reads_views_by_their_strides(layout):
    q, caches, scales, tables, sl = _inputs([300, 77], 4, 8, 2, 64, 32, BF16, E4M3, seed=5)
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl)
    both = torch.stack([c.view(torch.uint8) for c in caches], 1)  # [P, 2, page, Hkv, D]
    if layout == "hnd":
        both = both.transpose(2, 3).contiguous().transpose(2, 3)
    both = both.cuda().view(E4M3) if layout != "hnd" else \
        both.transpose(2, 3).contiguous().cuda().view(E4M3).transpose(2, 3)
    ks, vs = torch.stack(scales, 1).cuda().unbind(1) if layout == "scales_together" \
        else _cuda(*scales)
    qc, bt, slc = _cuda(q, tables, sl)
    out = torch.full_like(qc, 7.0)
    got = paged_attention_scaled(qc, both[:, 0], both[:, 1], ks, vs, bt, slc, out=out)
    assert got.data_ptr() == out.data_ptr()
    ref.assert_within(out, want, bound)


def test_attention_softmax_and_output_scale():
    q, caches, scales, tables, sl = _inputs([129], 4, 4, 1, 128, 16, F16, E4M3, seed=6)
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl, scale=0.25, out_scale=-1.5)
    out = paged_attention_scaled(*_cuda(q, *caches, *scales, tables, sl), scale=0.25,
                                 out_scale=-1.5)
    ref.assert_within(out, want, bound)


# ----- append -----


def _append_case(lens, new, q_len, hkv, d, page, dtype, kv, seed=0):
    g = torch.Generator().manual_seed(seed)
    pool = sum(-(-max(n, 0) // page) for n in lens) + 2
    tables, free = _tables(lens, page, pool, g)
    x = [torch.randn(len(lens), q_len, hkv, d, generator=g) for _ in range(2)]
    for t in x:  # sizes that differ from token to token, so that scales grow and do not
        t.mul_(2.0 ** torch.randint(-4, 4, (len(lens), q_len, hkv, 1), generator=g))
    key, value = (t.to(dtype) for t in x)
    caches, scales = [], []
    for _ in range(2):
        codes, scale = ref.quantise(torch.randn(pool, page, hkv, d, generator=g), kv)
        caches.append(codes)
        scales.append(scale)
    sl = torch.tensor(lens, dtype=torch.int32)
    nl = None if new is None else torch.tensor(new, dtype=torch.int32)
    return key, value, caches, scales, tables, sl, nl


def _check_append(key, value, caches, scales, tables, sl, nl):
    gc = [c.cuda() for c in caches]
    gs = [s.cuda() for s in scales]
    append_scaled_kv(key.cuda(), value.cuda(), *gc, *gs, tables.cuda(), sl.cuda(),
                     new_lens=None if nl is None else nl.cuda())
    want = [c.clone() for c in caches]
    ws = [s.clone() for s in scales]
    ties = ref.append(key, value, want, ws, tables, sl, nl)
    for g, w, s, v, tie in zip(gc, want, gs, ws, ties):
        assert torch.equal(s.cpu(), v)
        a, b = g.cpu().view(torch.uint8), w.view(torch.uint8)
        if g.dtype is E4M3:  # a NaN's sign says nothing
            a, b = (torch.where((t & 0x7F) == 0x7F, 0x7F, t) for t in (a, b))
        assert not ((a != b) & ~tie).any()
        # Beside a border the neighbouring code is right too, and nothing else.
        off = (g.cpu().float() - w.float()).abs()
        step = 1.0 if g.dtype is INT8 else w.float().abs() / 8 + 2.0 ** -9
        assert ((off <= step) | ~tie).all() and tie.float().mean() < 0.02
    return gc, gs


@pytest.mark.parametrize("kv", [E4M3, INT8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("page,d,hkv", [(16, 128, 8), (16, 64, 3), (32, 256, 2), (64, 128, 5),
                                        (128, 64, 1), (128, 256, 2), (256, 128, 2),
                                        (256, 256, 1)])
def test_append_blocks(page, d, hkv, dtype, kv):
    """From the middle of a page, over whole pages, into a last one; one token; none."""
    lens = [3 * page + 5, page, 1, page + 1, 7, 2 * page - 1, 0]
    new = [2 * page + 9, page, 1, 1, 0, 3, 0]
    _check_append(*_append_case(lens, new, 2 * page + 9, hkv, d, page, dtype, kv, seed=page + d))


@pytest.mark.parametrize("q_len", [1, 2, 4, 16, 17])
def test_append_every_sequence_q_tokens(q_len):
    _check_append(*_append_case([q_len, 100, 33, 16 * 9 + 1, 16 * 5], None, q_len, 4, 128, 16,
                                BF16, E4M3, seed=q_len))


def test_append_lengths_outside_their_range():
    """More new tokens than the call brings or the sequence holds, negative counts."""
    case = list(_append_case([5, 40, 20, 33], [9, 99, -3, 2], 8, 2, 64, 16, F16, INT8, seed=1))
    _check_append(*case)
    case[5] = torch.tensor([-4, 40, 20, 33], dtype=torch.int32)
    _check_append(*case)


def test_append_leaves_out_pages_that_are_not_there():
    key, value, caches, scales, tables, sl, nl = _append_case(
        [40, 40, 40], None, 20, 2, 64, 16, F16, E4M3, seed=2)
    tables[0, 2], tables[1, 1] = -1, caches[0].shape[0]
    _check_append(key, value, caches, scales, tables, sl, nl)
    _check_append(key, value, caches, scales, tables[:, :2].contiguous(), sl, nl)


@pytest.mark.parametrize("kv", [E4M3, INT8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_append_zeros_infinities_and_nan(dtype, kv):
    key, value, caches, scales, tables, sl, nl = _append_case(
        [35, 16, 20], None, 16, 2, 64, 16, dtype, kv, seed=7)
    key[0] = 0.0                 # a fresh page of zeros, and a page that keeps its scale
    value[1] = 0.0
    value[1, 3, 0, 4] = float("nan")
    key[1, 2, 1, 5], key[1, 9, 1, 6] = float("inf"), -float("inf")
    key[2, 5, 0, 7] = float("nan")
    value[2] = torch.finfo(dtype).smallest_normal * 3
    gc, gs = _check_append(key, value, caches, scales, tables, sl, nl)
    assert all(torch.isfinite(s).all() for s in gs)


def test_append_reads_strided_tokens():
    """K and V as slices of one projection's output, and caches and scales interleaved."""
    key, value, caches, scales, tables, sl, nl = _append_case(
        [70, 21], [33, 4], 40, 2, 64, 32, F16, E4M3, seed=8)
    both = torch.cat([key, value], 2).transpose(0, 1).contiguous().cuda().transpose(0, 1)
    pool = torch.stack([c.view(torch.uint8) for c in caches], 1).cuda().view(E4M3)
    sc = torch.stack(scales, 1).cuda()
    append_scaled_kv(both[:, :, :2], both[:, :, 2:], pool[:, 0], pool[:, 1], sc[:, 0], sc[:, 1],
                     tables.cuda(), sl.cuda(), new_lens=nl.cuda())
    gc, gs = _check_append(key, value, caches, scales, tables, sl, nl)
    assert torch.equal(pool[:, 0].view(torch.uint8), gc[0].view(torch.uint8))
    assert torch.equal(pool[:, 1].view(torch.uint8), gc[1].view(torch.uint8))
    assert torch.equal(sc[:, 0], gs[0]) and torch.equal(sc[:, 1], gs[1])


def test_append_then_attend():
    """A prompt in chunks, then draft tokens with some taken back: what attention reads is
    what the last append of every slot left."""
    g = torch.Generator().manual_seed(9)
    b, hkv, d, page, total = 3, 2, 128, 16, 210
    k, v = (torch.randn(b, total, hkv, d, generator=g).half() for _ in range(2))
    pool = 3 * b * 5
    tables = torch.randperm(pool, generator=g)[:b * 14].view(b, 14).to(torch.int32)
    caches = [torch.zeros(pool, page, hkv, d, dtype=E4M3, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pool, hkv, device="cuda") for _ in range(2)]
    cc = [c.cpu() for c in caches]
    cs = [s.cpu() for s in scales]
    bt = tables.cuda()
    at = torch.zeros(b, dtype=torch.int32)
    for n in ([90, 1, 16], [40, 100, 17], [4, 4, 4], [4, 4, 4], [1, 4, 2]):
        n = torch.tensor(n, dtype=torch.int32)
        q_len = int(n.max())
        rows = torch.minimum(at[:, None] + torch.arange(q_len), torch.tensor(total - 1)).long()
        key, value = (x[torch.arange(b)[:, None], rows] for x in (k, v))
        at += n
        append_scaled_kv(key.cuda(), value.cuda(), *caches, *scales, bt, at.cuda(),
                         new_lens=n.cuda())
        ref.append(key, value, cc, cs, tables, at, n)
        if q_len == 4:
            q = torch.randn(b, 4, 8, d, generator=g).half()
            want, bound, _ = ref.attention(q, *[c.cpu() for c in caches],
                                           *[s.cpu() for s in scales], tables, at)
            out = paged_attention_scaled(q.cuda(), *caches, *scales, bt, at.cuda())
            ref.assert_within(out, want, bound)
            at -= torch.tensor([3, 1, 2], dtype=torch.int32)  # draft tokens not accepted
    for g_, w in zip(scales, cs):
        assert torch.equal(g_.cpu(), w)
