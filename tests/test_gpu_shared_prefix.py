"""Attention over shared prefixes on the GPU, against a plain statement in 64 bits."""

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd.masks import pack_draft_mask  # noqa: E402
from small_q_attention_amd.shared_prefix import (paged_attention_shared_prefix,  # noqa: E402
                                                 plan_shared_prefix)
from tests import _part_reference as ref  # noqa: E402
from tests._part_reference import BF16, E4M3, F16, INT8  # noqa: E402

pytestmark = pytest.mark.gpu

CACHES = [(F16, None, False), (BF16, None, False), (F16, E4M3, False), (BF16, E4M3, False),
          (F16, E4M3, True), (BF16, INT8, True)]


def inputs(groups, lens, q_len, hq, hkv, d, page, dtype, kv, scaled, seed=0, width=None):
    """``lens`` are whole lengths. Only the group's first sequence that is long enough names
    the shared pages; the others' entries there are -1, as are those past a length."""
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    own = [0] * b
    leader = [None] * b
    for first, count, pages in groups:
        able = [i for i in range(first, first + count) if lens[i] - q_len >= pages * page]
        if count > 1 and pages > 0:
            for i in able:
                own[i], leader[i] = pages, able[0]
    used = [-(-max(n, 0) // page) for n in lens]
    pool = sum(used) + 3
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    tables = torch.full((b, width or max(used + [max([p for *_, p in groups] + [1])])), -1,
                        dtype=torch.int32)
    full = tables.clone()
    at = 0
    for i in range(b):
        start = 0 if leader[i] in (None, i) else own[i]
        tables[i, start:used[i]] = full[i, start:used[i]] = perm[at:at + used[i] - start]
        if start:
            full[i, :start] = full[leader[i], :start]
        at += used[i] - start
    q = torch.randn(b, q_len, hq, d, generator=g).to(dtype)
    caches, scales = zip(*(ref.cache(pool, page, hkv, d, dtype, kv, scaled, g) for _ in range(2)))
    for c, s in zip(caches, scales):
        ref.spoil(c, perm[at:].long())
        for i, n in enumerate(lens):
            if n > 0 and n % page:
                ref.spoil(c, int(full[i, n // page]), torch.arange(n % page, page))
    return q, list(caches), list(scales), tables, full, torch.tensor(lens, dtype=torch.int32)


def p_step(dtype, scaled):
    """Probabilities of the shared pages may be rounded once to the query's type."""
    return 2.0 ** -9 if dtype is BF16 and not scaled else 2.0 ** -11


def check(groups, lens, q_len, hq, hkv, d, page, dtype, kv, scaled, seed=0, tree=None, **kw):
    q, caches, scales, tables, full, sl = inputs(groups, lens, q_len, hq, hkv, d, page, dtype, kv,
                                                 scaled, seed, **kw)
    want, bound = ref.attention(
        q, *caches, *scales, full, sl,
        lambda i, n: ref.window_seen(n, q_len, 1 << 30, 0, None if tree is None else tree[i]),
        p_step=p_step(dtype, scaled))
    qc, kc, vc, ks, vs, bt, slc = ref.cuda(q, *caches, *scales, tables, sl)
    mask = None if tree is None else pack_draft_mask(tree).cuda()
    plan = plan_shared_prefix(groups, len(lens), q_len, hq, hkv, d, page)
    outs = []
    for most in (0, max(max(lens), 1)):
        out = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, key_scale=ks,
                                            value_scale=vs, max_seq_len=most, mask=mask)
        ref.assert_within(out, want, bound, f"max_seq_len {most}")
        outs.append(out)
    again = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, key_scale=ks, value_scale=vs,
                                          mask=mask)
    assert torch.equal(outs[0], again)


@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
@pytest.mark.parametrize("count", [2, 5, 9, 17, 40])
def test_one_group(dtype, kv, scaled, count):
    """4 to 640 rows of a kv head over 500 shared tokens: blocks of every size."""
    lens = [512 + 3 + (29 * i) % 130 for i in range(count)]
    check([(0, count, 32)], lens, 3, 8, 2, 128, 16, dtype, kv, scaled, seed=count)


@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
@pytest.mark.parametrize("q_len,hq,hkv,d,page", [
    (1, 8, 8, 128, 16), (1, 32, 8, 128, 32), (16, 16, 4, 128, 64), (7, 15, 3, 128, 256),
    (5, 5, 5, 64, 16), (1, 8, 1, 64, 64), (8, 32, 4, 64, 32), (2, 16, 2, 256, 16),
    (8, 8, 2, 256, 128), (16, 4, 4, 64, 16)])
def test_shapes(dtype, kv, scaled, q_len, hq, hkv, d, page):
    pages = 512 // page
    lens = [512 + n for n in (16, 33, 70, 17, 100, 260)]
    check([(0, 2, pages), (2, 4, pages // 2)], lens, q_len, hq, hkv, d, page, dtype, kv, scaled,
          seed=q_len)


@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
def test_groups_of_many_kinds(dtype, kv, scaled):
    """Sequences of no group, groups of one sequence, of no pages, of one page, of many;
    padded and short sequences inside groups, the first of a group among them."""
    page, q = 16, 2
    groups = [(1, 3, 4), (4, 1, 9), (5, 2, 0), (8, 6, 33), (14, 2, 1)]
    lens = [100, 64 + 2, 64 + 30, 64 + 1, 200, 31, 18, 5,
            0, 528 + 2, 528 + 40, 300, 528 + 1, 528 + 77, 16, 18, 1]
    check(groups, lens, q, 8, 2, 128, page, dtype, kv, scaled, seed=2)


@pytest.mark.parametrize("dtype,kv,scaled", CACHES[:3])
def test_nobody_reaches_past_the_shared_pages(dtype, kv, scaled):
    check([(0, 3, 20)], [0, 40, 321], 2, 8, 2, 64, 16, dtype, kv, scaled)
    check([], [30, 40, 321], 2, 8, 2, 64, 16, dtype, kv, scaled)


@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
def test_draft_trees(dtype, kv, scaled):
    lens = [256 + 4, 256 + 20, 256 + 5, 256 + 300, 4]
    tree = ref.trees(len(lens), 4, seed=3, empty=(0,))
    check([(0, 5, 16)], lens, 4, 8, 2, 128, 16, dtype, kv, scaled, seed=5, tree=tree)


@pytest.mark.parametrize("pages", [1, 2, 3, 5, 7, 31, 127, 260])
@pytest.mark.parametrize("count", [3, 60])
def test_shared_lengths(pages, count):
    lens = [pages * 16 + 4 + i % 7 for i in range(count)]
    check([(0, count, pages)], lens, 4, 8, 2, 128, 16, F16, None, False, seed=pages)
    check([(0, count, pages)], lens, 2, 4, 2, 64, 16, BF16, E4M3, False, seed=pages)


def test_the_result_is_attention_over_the_whole_tables():
    from small_q_attention_amd.cuda import paged_mtp_attention

    lens = [2048 + 8 + 5 * i for i in range(12)]
    q, (k, v), _, _, full, sl = inputs([(0, 12, 128)], lens, 8, 32, 8, 128, 16, F16, None, False)
    full = full.clamp(min=0)
    qc, kc, vc, bt, slc = ref.cuda(q, k, v, full, sl)
    plan = plan_shared_prefix([(0, 12, 128)], 12, 8, 32, 8, 128, 16)
    a = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan)
    b = paged_mtp_attention(qc, kc, vc, bt, slc)
    assert (a.float() - b.float()).abs().max() <= 2e-3


@pytest.mark.parametrize("dtype,kv", [(F16, None), (BF16, None), (F16, E4M3)])
def test_values_that_are_not_finite(dtype, kv):
    """NaN in a shared token reaches every row that shares it, in its dimension; one in a
    draft token the rows that see it."""
    q_len, page, lens = 4, 16, [256 + 40, 256 + 9, 200, 256 + 21]
    q, (k, v), _, tables, full, sl = inputs([(0, 4, 16)], lens, q_len, 8, 2, 128, page, dtype, kv,
                                            False)

    def put(c, i, t, h, e):
        raw = c.view(torch.uint8) if c.element_size() == 1 else c
        raw[int(full[i, t // page]), t % page, h, e] = 0x7F if c.element_size() == 1 \
            else float("nan")

    put(v, 0, 100, 1, 9)
    put(v, 1, 256 + 9 - 3, 0, 3)
    put(k, 3, 256 + 21 - 2, 1, 0)
    put(k, 2, 50, 0, 0)
    want, bound = ref.attention(q, k, v, None, None, full, sl,
                                lambda i, n: ref.window_seen(n, q_len, 1 << 30, 0),
                                p_step=p_step(dtype, False))
    qc, kc, vc, bt, slc = ref.cuda(q, k, v, tables, sl)
    plan = plan_shared_prefix([(0, 4, 16)], 4, q_len, 8, 2, 128, page)
    ref.assert_within(paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan), want, bound)


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("kv", [None, E4M3])
def test_interleaved_caches(layout, kv):
    lens, q_len, hkv, d, page = [300, 277, 290] * 10, 4, 4, 128, 32
    q, (k, v), _, tables, full, sl = inputs([(0, 30, 8)], lens, q_len, 16, hkv, d, page, F16, kv,
                                            False)
    want, bound = ref.attention(q, k, v, None, None, full, sl,
                                lambda i, n: ref.window_seen(n, q_len, 1 << 30, 0))
    raw = [c.view(torch.uint8) if kv else c for c in (k, v)]
    if layout == "HND":
        raw = [c.transpose(1, 2) for c in raw]
    both = torch.stack(raw, 1).contiguous().cuda()
    both = both.view(kv) if kv else both
    views = [both[:, 0], both[:, 1]]
    if layout == "HND":
        views = [c.transpose(1, 2) for c in views]
    qc, bt, slc = ref.cuda(q, tables, sl)
    plan = plan_shared_prefix([(0, 30, 8)], 30, q_len, 16, hkv, d, page)
    ref.assert_within(paged_attention_shared_prefix(qc, *views, bt, slc, plan), want, bound)


def test_scales_out_and_workspace():
    lens = [512 + 30, 512 + 700]
    q, (k, v), _, tables, full, sl = inputs([(0, 2, 32)], lens, 4, 8, 2, 128, 16, F16, None, False)
    want, bound = ref.attention(q, k, v, None, None, full, sl,
                                lambda i, n: ref.window_seen(n, 4, 1 << 30, 0), scale=0.05,
                                out_scale=-1.5)
    qc, kc, vc, bt, slc = ref.cuda(q, k, v, tables, sl)
    plan = plan_shared_prefix([(0, 2, 32)], 2, 4, 8, 2, 128, 16)
    out = torch.empty_like(qc)
    ws = torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")
    got = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, scale=0.05, out_scale=-1.5,
                                        out=out, workspace_buffer=ws)
    assert got is out
    ref.assert_within(out, want, bound)
    with pytest.raises(ValueError, match="workspace_buffer"):
        paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, workspace_buffer=ws[:64])


def test_lengths_past_the_table_and_ids_outside_the_pool():
    """As for the other attention calls: held to the table's pages, page 0 in their place."""
    q, (k, v), _, _, full, sl = inputs([(0, 3, 2)], [64, 64, 64], 2, 4, 2, 64, 16, F16, None,
                                       False)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    qc, kc, vc, bt, _ = ref.cuda(q, k, v, full, sl)
    plan = plan_shared_prefix([(0, 3, 2)], 3, 2, 4, 2, 64, 16)
    for n in (65, 10**6, 2**31 - 1, -5):
        lens = torch.tensor([n, 64, 64], dtype=torch.int32, device="cuda")
        out = paged_attention_shared_prefix(qc, kc, vc, bt, lens, plan)
        assert torch.isfinite(out).all()
        assert n > 0 or not out[0].any()
    lens = torch.tensor([64, 64, 64], dtype=torch.int32, device="cuda")
    bad, zero = bt.clone(), bt.clone()
    bad[0], zero[0] = 10**6, 0
    assert torch.equal(paged_attention_shared_prefix(qc, kc, vc, bad, lens, plan),
                       paged_attention_shared_prefix(qc, kc, vc, zero, lens, plan))
