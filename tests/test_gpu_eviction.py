"""Attention weights added up and eviction by them, on the GPU, against plain statements in
64 bits."""

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd.eviction import (accumulate_attention_weights,  # noqa: E402
                                            evict_by_weight)
from small_q_attention_amd.masks import pack_draft_mask  # noqa: E402
from small_q_attention_amd.scaled_cache import (append_scaled_kv,  # noqa: E402
                                                paged_attention_scaled)
from tests import _cache_reference as ref  # noqa: E402
from tests.test_gpu_scaled_cache import _cuda, _inputs, _tables, _trees  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3, INT8, F16, BF16 = torch.float8_e4m3fn, torch.int8, torch.float16, torch.bfloat16
TYPES = [(F16, F16, False), (BF16, BF16, False), (F16, E4M3, True), (BF16, INT8, True),
         (BF16, E4M3, True), (F16, INT8, True), (F16, E4M3, False)]
IDS = ["fp16", "bf16", "fp16-e4m3s", "bf16-int8s", "bf16-e4m3s", "fp16-int8s", "fp16-e4m3"]


def _weigh_inputs(lens, q_len, hq, hkv, d, page, dtype, kv, scaled, seed, width=None):
    coded = kv if scaled else E4M3
    q, caches, scales, tables, sl = _inputs(lens, q_len, hq, hkv, d, page, dtype, coded, seed, width)
    k, ks = caches[0], scales[0]
    if not scaled:
        ks = None
        if kv is E4M3:  # codes as they are
            q = (q.float() / 64).to(dtype)
        else:
            x = k.float() / 100  # unowned slots stay NaN
            k = x.to(kv)
    g = torch.Generator().manual_seed(seed + 1)
    weights = torch.rand(len(lens), hkv, max(max(lens), 1) + 7, generator=g)
    return q, k, ks, tables, sl, weights


def _check_weigh(lens, q_len, hq, hkv, d, page, types, seed=0, trees=None, width=None, cut=0):
    q, k, ks, tables, sl, weights = _weigh_inputs(lens, q_len, hq, hkv, d, page, *types, seed,
                                                  width)
    if cut:
        weights = weights[:, :, :cut].contiguous()
    _, _, mass = ref.attention(q, k, None, ks, None, tables, sl, trees)
    want, bound = ref.weights_after(weights, mass, sl, q_len)
    mask = None if trees is None else pack_draft_mask(trees).cuda()
    args = _cuda(q, k, tables, sl)
    ksc = None if ks is None else ks.cuda()
    results = []
    for most in (0, max(max(lens), 1), 0):
        got = weights.cuda()
        out = accumulate_attention_weights(*args, got, key_scale=ksc, max_seq_len=most, mask=mask)
        assert out is got
        ref.assert_within(got, want, bound, f"max_seq_len {most}")
        results.append(got)
    assert torch.equal(results[0], results[2])


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("q_len,group", [(1, 1), (1, 4), (4, 4), (5, 3), (8, 4), (9, 7)])
def test_weights_rows(q_len, group, types):
    """Few rows (the scores go through memory) and many (K is read twice)."""
    _check_weigh([777, 41, 2048, q_len], q_len, 4 * group, 4, 128, 16, types, seed=q_len)


@pytest.mark.parametrize("types", TYPES[:4], ids=IDS[:4])
@pytest.mark.parametrize("d,q_len", [(64, 1), (64, 4), (64, 16), (256, 1), (256, 5), (256, 8)])
def test_weights_head_dims(d, q_len, types):
    _check_weigh([1500, 17, 333], q_len, 16, 4, d, 32, types, seed=d)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("hkv", [1, 2, 3, 5, 8])
def test_weights_pages_and_heads(page, hkv):
    _check_weigh([1111, 256, 255, 1], 2, 4 * hkv, hkv, 128, page, TYPES[0], seed=page + hkv)


@pytest.mark.parametrize("q_len", [3, 8])
@pytest.mark.parametrize("lens", [[0], [1], [2], [15, 16, 17], [0, 0], [64, 65, 0, 1], [5000],
                                  [3] * 70, [33 * (i % 9) for i in range(300)]])
def test_weights_lengths(lens, q_len):
    _check_weigh(lens, q_len, 8, 2, 64, 16, TYPES[0], seed=len(lens),
                 width=max(max(lens) // 16 + 2, 3))


@pytest.mark.parametrize("q_len", [2, 9])
@pytest.mark.parametrize("b", [65, 128, 300, 530])
def test_weights_batches_about_as_large_as_the_chip(b, q_len):
    """Few work items to spare, and none (eight kv heads: 512 and 256 items)."""
    lens = [(37 * i * i) % 300 for i in range(b)]
    lens[b // 3] = 5000
    _check_weigh(lens, q_len, 8, 8, 64, 16, TYPES[2], seed=b)


@pytest.mark.parametrize("types", [TYPES[0], TYPES[3]], ids=[IDS[0], IDS[3]])
@pytest.mark.parametrize("q_len", [1, 6, 16])
def test_weights_draft_trees(q_len, types):
    lens = [600, q_len, 33 + q_len, q_len + 1]
    _check_weigh(lens, q_len, 8, 2, 128, 16, types, seed=q_len, trees=_trees(4, q_len, 1, (0, 3)))


@pytest.mark.parametrize("types", [TYPES[0], TYPES[3]], ids=[IDS[0], IDS[3]])
def test_weights_of_a_wide_table(types):
    """A table whose scores would pass 1 GiB: few rows, and K is read twice all the same."""
    _check_weigh([700, 33], 2, 16, 4, 128, 16, types, seed=8, width=(1 << 18) + 5)


@pytest.mark.parametrize("q_len", [2, 12])
def test_weights_narrower_than_the_sequences(q_len):
    _check_weigh([300, 40], q_len, 8, 2, 128, 16, TYPES[1], cut=45)


@pytest.mark.parametrize("q_len", [2, 12])
def test_weights_nan_keys(q_len):
    """A NaN key makes NaN every weight of the head that a row seeing it gives, and none
    where a row does not see the token."""
    q, k, ks, tables, sl, weights = _weigh_inputs([70, 33], q_len, 8, 2, 128, 16, F16, F16, False, 5)
    k[int(tables[0, 69 // 16]), 69 % 16, 1, 3] = float("nan")  # the last draft token
    _, _, mass = ref.attention(q, k, None, None, None, tables, sl)
    want, bound = ref.weights_after(weights, mass, sl, q_len)
    assert torch.isnan(want[0, 1, :70]).all() and torch.isnan(want).sum() == 70
    got = accumulate_attention_weights(*_cuda(q, k, tables, sl, weights))
    ref.assert_within(got, want, bound)


def test_weights_strided_and_added_up():
    """Calls that follow each other: a draft, taken back in part, and the next one."""
    q, k, ks, tables, sl, _ = _weigh_inputs([200, 77], 4, 8, 2, 128, 16, F16, INT8, True, 6)
    store = torch.full((2, 5, 300), 0.5)
    want = store[:, 1:3, 10:260]
    got = store.clone().cuda()
    view = got[:, 1:3, 10:260]
    for lens in ([190, 60], [192, 64], [195, 64]):
        sl = torch.tensor(lens, dtype=torch.int32)
        _, _, mass = ref.attention(q, k, None, ks, None, tables, sl)
        want, bound = ref.weights_after(want, mass, sl, 4)
        accumulate_attention_weights(*_cuda(q, k, tables, sl), view, key_scale=ks.cuda())
        ref.assert_within(view, want, 3 * bound)
    rest = torch.ones_like(store, dtype=torch.bool)
    rest[:, 1:3, 10:260] = False
    assert (got.cpu()[rest] == 0.5).all()


# ----- eviction -----


def _evict_case(lens, hkv, d, page, kv, budget, seed=0, ties=False):
    g = torch.Generator().manual_seed(seed)
    scaled = kv in (E4M3, INT8)
    _, caches, scales, tables, sl = _inputs(lens, 1, hkv, hkv, d, page, F16, kv if scaled else E4M3,
                                            seed)
    if not scaled:
        caches = [c.float().to(kv) for c in caches]
        scales = None
    weights = torch.rand(len(lens), hkv, max(max(lens), 1) + 5, generator=g)
    if ties:
        weights = (weights * 4).floor() / 4
        weights[:, :, ::7] = -0.0
    used = [min(max(n, 0), budget) for n in lens]
    new_tables, _ = _tables(used, page, sum(-(-n // page) for n in used) + 1, g,
                            width=-(-budget // page))
    pages = int(sum(-(-n // page) for n in used)) + 1
    fill = torch.full((pages, page, hkv, d), 3.0)
    into = [fill.clone().to(kv) for _ in range(2)]
    into_scales = [torch.full((pages, hkv), 9.0) for _ in range(2)] if scaled else None
    return weights, caches, scales, tables, sl, new_tables, into, into_scales


def _same(a, b):
    a, b = a.cpu(), b
    if a.element_size() == 1:
        a, b = a.view(torch.uint8), b.view(torch.uint8)
    elif a.dtype in (F16, BF16):
        a, b = a.view(torch.int16), b.view(torch.int16)
    return torch.equal(a, b)


def _check_evict(case, budget, sink, recent, in_place=False):
    weights, caches, scales, tables, sl, new_tables, into, into_scales = case
    gi = [x.cuda() for x in into]
    gs = [None, None] if scales is None else [x.cuda() for x in into_scales]
    src = [None, None] if scales is None else _cuda(*scales)
    w = weights.cuda()
    lens, nw, kept = evict_by_weight(
        w, *_cuda(*caches, tables, sl, new_tables), budget, sink=sink, recent=recent,
        key_scale=src[0], value_scale=src[1], into=(*gi, *gs), new_weights=w if in_place else None)
    want = ref.evict(weights, caches, scales, tables, sl, new_tables, budget, sink, recent, into,
                     into_scales)
    assert torch.equal(lens.cpu(), want[0])
    assert torch.equal(kept.cpu(), want[2])
    if in_place:
        assert nw.data_ptr() == w.data_ptr() and (nw[:, :, budget:] == 0).all()
        nw = nw[:, :, :budget]
    else:
        assert torch.equal(w.cpu().nan_to_num(), weights.nan_to_num())
    assert torch.equal(nw.cpu().nan_to_num(nan=-7.0), want[1].nan_to_num(nan=-7.0))
    for a, b in zip(gi, into):
        assert _same(a, b)
    if scales is not None:
        for a, b in zip(gs, into_scales):
            assert torch.equal(a.cpu(), b)


KINDS = [F16, BF16, E4M3, INT8]
KIND_IDS = ["fp16", "bf16", "e4m3", "int8"]


@pytest.mark.parametrize("kv", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("page,d,hkv", [(16, 128, 8), (32, 64, 3), (64, 256, 1), (256, 128, 2)])
def test_evict_layouts(page, d, hkv, kv):
    lens = [700, 100, 99, 101, 5, 0, 333]
    _check_evict(_evict_case(lens, hkv, d, page, kv, 100, seed=page), 100, 4, 17)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (16, 0, 0),
                                                (50, 25, 25), (50, 0, 50), (63, 3, 9),
                                                (1025, 0, 1), (1500, 64, 300)])
def test_evict_budgets(budget, sink, recent, in_place):
    _check_evict(_evict_case([1, 64, 1024, 1026, 2500], 2, 64, 16, F16, budget, seed=budget),
                 budget, sink, recent, in_place)


@pytest.mark.parametrize("budget", [7, 100, 600])
def test_evict_ties_go_to_the_earlier_token(budget):
    case = _evict_case([1000, 3000, 777], 2, 64, 16, BF16, budget, seed=3, ties=True)
    case[0][2] = 0.25  # all alike
    case[0][2, 1, ::2] = -0.0
    case[0][2, 1, 1::2] = 0.0
    _check_evict(case, budget, 2, 3)


def test_evict_weights_that_are_not_numbers():
    case = _evict_case([500, 500, 500], 2, 64, 16, F16, 90, seed=4)
    w = case[0]
    w[0, 0, 10:480:3] = float("nan")
    w[0, 1] = float("nan")
    w[1, 0, ::5] = float("inf")
    w[1, 1, ::2] = -float("inf")
    w[2, 0] = -w[2, 0]
    w[2, 1] *= 2.0 ** -140  # subnormal
    _check_evict(case, 90, 5, 6)


def test_evict_a_long_sequence():
    _check_evict(_evict_case([70001, 12], 1, 64, 64, E4M3, 5001, seed=5), 5001, 10, 100)


def test_evict_long_sequences_in_place():
    """Weights too many to be held: they move over themselves."""
    _check_evict(_evict_case([40001, 33000, 12], 1, 64, 64, E4M3, 5001, seed=6, ties=True), 5001,
                 10, 100, True)


def test_evict_within_one_pool():
    """New pages of the same pool, and pages two sequences share among the old ones."""
    weights, caches, scales, tables, sl, _, _, _ = _evict_case([300, 300], 2, 128, 16, E4M3, 64,
                                                               seed=6)
    tables[1, :5] = tables[0, :5]
    n = caches[0].shape[0]
    caches = [torch.cat([c.view(torch.uint8), torch.zeros(9, *c.shape[1:], dtype=torch.uint8)])
              .view(E4M3) for c in caches]
    scales = [torch.cat([s, torch.zeros(9, 2)]) for s in scales]
    new_tables = (n + torch.randperm(8, generator=torch.Generator().manual_seed(1))).view(2, 4) \
        .to(torch.int32)
    gc, gs = _cuda(*caches), _cuda(*scales)
    lens, nw, kept = evict_by_weight(weights.cuda(), *gc, *_cuda(tables, sl, new_tables), 64,
                                     recent=8, key_scale=gs[0], value_scale=gs[1])
    want = ref.evict(weights, caches, scales, tables, sl, new_tables, 64, 0, 8, caches, scales)
    assert torch.equal(kept.cpu(), want[2]) and torch.equal(nw.cpu(), want[1])
    for a, b in zip(gc + gs, caches + scales):
        assert _same(a, b) or torch.equal(a.cpu().nan_to_num(), b.nan_to_num())


def test_evict_leaves_out_pages_that_are_not_there():
    case = list(_evict_case([200, 200], 2, 64, 16, F16, 48, seed=7))
    case[5][0, 1], case[5][1, 2] = -1, case[6][0].shape[0]
    weights, caches, _, tables, sl, new_tables, into, _ = case
    gi = _cuda(*into)
    evict_by_weight(weights.cuda(), *_cuda(*caches, tables, sl, new_tables), 48, into=tuple(gi))
    tables_ok = new_tables.clone()
    spare = into[0].shape[0]
    tables_ok[0, 1], tables_ok[1, 2] = spare, spare
    wide = [torch.cat([x, x[:1]]) for x in into]
    ref.evict(weights, caches, None, tables, sl, tables_ok, 48, 0, 0, wide, None)
    for a, b in zip(gi, wide):
        assert _same(a, b[:spare])


@pytest.mark.parametrize("kv", [E4M3, INT8], ids=["e4m3", "int8"])
def test_a_decoding_loop(kv):
    """Prompt, draft steps, weights, eviction, further steps on the new pages: every stage
    against the plain statement of the same state."""
    g = torch.Generator().manual_seed(8)
    b, q_len, hq, hkv, d, page, budget = 3, 4, 8, 2, 128, 16, 80
    pool = 80
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    tables, new_tables = perm[:42].view(b, 14), perm[42:42 + 21].view(b, 7)
    caches = [torch.zeros(pool, page, hkv, d, dtype=kv, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pool, hkv, device="cuda") for _ in range(2)]
    weights = torch.zeros(b, hkv, 14 * page, device="cuda")
    lens = torch.tensor([150, 64, 101], dtype=torch.int32)
    key, value = (torch.randn(b, 150, hkv, d, generator=g).half().cuda() for _ in range(2))
    bt = tables.cuda()
    append_scaled_kv(key, value, *caches, *scales, bt, lens.cuda(), new_lens=lens.cuda())
    for step in range(6):
        if step == 3:
            before = [x.cpu() for x in (*caches, *scales, weights)]
            out = evict_by_weight(weights, *caches, bt, lens.cuda(), new_tables.cuda(), budget,
                                  sink=2, recent=9, key_scale=scales[0], value_scale=scales[1],
                                  new_weights=weights)
            want = ref.evict(before[4], before[:2], before[2:4], tables, lens, new_tables, budget,
                             2, 9, before[:2], before[2:4])
            assert torch.equal(out[0].cpu(), want[0]) and torch.equal(out[2].cpu(), want[2])
            for a, w in zip((*caches, *scales), before[:4]):
                assert _same(a, w) if a.element_size() == 1 else torch.equal(a.cpu(), w)
            lens, tables, bt = out[0].cpu(), new_tables, new_tables.cuda()
        lens = lens + q_len - (step % 3 if step not in (0, 3) else 0)
        q, k, v = (torch.randn(b, q_len, n, d, generator=g).half() for n in (hq, hkv, hkv))
        sl = lens.cuda()
        append_scaled_kv(k.cuda(), v.cuda(), *caches, *scales, bt, sl)
        old = weights.cpu()
        out = paged_attention_scaled(q.cuda(), *caches, *scales, bt, sl)
        accumulate_attention_weights(q.cuda(), caches[0], bt, sl, weights, key_scale=scales[0])
        want, bound, mass = ref.attention(q, *[x.cpu() for x in (*caches, *scales)], tables, lens)
        ref.assert_within(out, want, bound, f"step {step}")
        want, bound = ref.weights_after(old, mass, lens, q_len)
        ref.assert_within(weights, want, bound, f"step {step}")


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,width,budget,sink,recent", [
    ([300, 64, 65, 5, 0], 64, 40, 3, 9),         # the recent tokens lie past the weights
    ([300, 120], 10, 100, 20, 7),                # so does the sink, and the budget
    ([500, 77], 1, 1, 0, 1),
    ([200, 3], 64, 64, 0, 0),                    # all weights fit, later tokens weigh 0
    ([9001, 4097, 4000, 12], 4000, 1000, 4, 100),  # longer than the registers' form holds
    ([70000, 33000], 33000, 5000, 4, 800),
])
def test_evict_sequences_longer_than_their_weights(lens, width, budget, sink, recent, in_place):
    """Tokens the weights do not reach weigh 0; the first and last ones stay as ever."""
    in_place = in_place and width >= budget  # else the buffer cannot hold the new weights
    case = list(_evict_case(lens, 2, 64, 16, E4M3, budget, seed=width, ties=width % 2 == 0))
    full = case[0]
    full[:, :, width:] = 0.0
    # Weights below 0 rank behind the tokens that have none.
    full[:, :, :width:5] *= -1.0
    case[0] = full[:, :, :width].contiguous()
    got = _evict_narrow(case, budget, sink, recent, in_place)
    want = ref.evict(full, *case[1:6], budget, sink, recent, *case[6:])
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert torch.equal(got[1][:, :, :budget], want[1]) and (got[1][:, :, budget:] == 0).all()
    for a, b in zip(got[3:], (*case[6], *case[7])):
        assert _same(a, b) or torch.equal(a, b)


def _evict_narrow(case, budget, sink, recent, in_place):
    weights, caches, scales, tables, sl, new_tables, into, into_scales = case
    w, ks, vs, bt, slc, nt, *moved = _cuda(weights, *scales, tables, sl, new_tables, *into,
                                           *into_scales)
    lens, nw, kept = evict_by_weight(w, *_cuda(*caches), bt, slc, nt, budget, sink=sink,
                                     recent=recent, key_scale=ks, value_scale=vs,
                                     into=tuple(moved), new_weights=w if in_place else None)
    return [x.cpu() for x in (lens, nw, kept, *moved)]


def test_evictions_in_turn_without_a_buffer_for_the_weights():
    """The weights that an eviction returns are as wide as its budget: of the tokens decoded
    after it the recent ones stay, whatever the weights do not say of them."""
    g = torch.Generator().manual_seed(12)
    b, hkv, d, page, budget, recent = 2, 2, 64, 16, 48, 20
    pool = torch.randn(64, page, hkv, d, generator=g).half()
    caches = [pool.cuda(), (pool * 2).cuda()]
    tables = torch.arange(2 * 8).view(2, 8).to(torch.int32)
    weights, lens = torch.rand(b, hkv, 128, generator=g), torch.tensor([120, 70], dtype=torch.int32)
    for step in range(3):
        new = (16 + 16 * step + torch.arange(2 * 8)).view(2, 8).to(torch.int32)
        full = torch.zeros(b, hkv, 128)
        full[:, :, :weights.shape[2]] = weights
        mine = [c.cpu() for c in caches]
        got = evict_by_weight(weights.cuda(), *caches, *_cuda(tables, lens, new), budget, sink=2,
                              recent=recent)
        want = ref.evict(full, mine, None, tables, lens, new, budget, 2, recent, mine, None)
        for a, w in zip(got, want):
            assert torch.equal(a.cpu(), w)
        for a, w in zip(caches, mine):
            assert _same(a, w)
        assert got[1].shape[2] == budget
        kept = got[2].cpu()
        assert (kept[:, :, -recent:] == lens[:, None, None] - recent + torch.arange(recent)).all()
        weights, tables, lens = got[1].cpu(), new, got[0].cpu() + torch.tensor([30, 17])
        lens = lens.to(torch.int32)
