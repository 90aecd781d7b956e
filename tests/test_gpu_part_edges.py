"""Attention over a window and over shared prefixes on the GPU where it is least alike to the
usual call: prefixes of very unlike lengths in one batch, partial rows past 32-bit offsets,
values that are not finite, plans dropped while their calls wait."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd import _lib, _op, scaled_cache, windowed  # noqa: E402,F401
from small_q_attention_amd.shared_prefix import (paged_attention_shared_prefix,  # noqa: E402
                                                 plan_shared_prefix)
from small_q_attention_amd.windowed import paged_attention_windowed  # noqa: E402
from tests import _part_reference as ref  # noqa: E402
from tests._part_reference import BF16, E4M3, F16, INT8  # noqa: E402
from tests.test_gpu_shared_prefix import inputs, p_step  # noqa: E402

pytestmark = pytest.mark.gpu

CACHES = [(F16, None, False), (BF16, None, False), (F16, E4M3, False), (BF16, E4M3, False),
          (F16, E4M3, True), (BF16, INT8, True)]


def everything(q_len):
    return lambda i, n: ref.window_seen(n, q_len, 1 << 30, 0)


def _copy(plan):
    p = _lib.SharedPlan()
    ctypes.memmove(ctypes.byref(p), ctypes.byref(plan), ctypes.sizeof(plan))
    return p


def _splits(pages, size):
    """As many splits of at most `size` pages as it takes, all alike."""
    return -(-pages // -(-pages // -(-pages // size))) if pages else 0


def _forge(monkeypatch, change):
    """Plans that ``change(plan, groups in 16-token pages)`` has altered; collects them."""
    real, made = _lib.plan_shared_prefix, []

    def forged(device, groups, shape, kv, most, width):
        plan, _, table = real(device, groups, shape, kv, most, width)
        plan = _copy(plan)
        change(plan, [(n, pages * (shape[5] // 16) * (n > 1)) for _, n, pages in groups])
        made.append(plan)
        return plan, int(_lib.load().sqa_shared_workspace_bytes(ctypes.byref(plan))), table

    monkeypatch.setattr(_lib, "plan_shared_prefix", forged)
    return made


# --------------------------------------------------------------------------------------
# Prefixes of very unlike lengths: the groups' partial rows lie packed.
# --------------------------------------------------------------------------------------

UNLIKE = [
    # A long one first, last and between short ones, groups of one and of no pages, sequences of
    # no group, some that do not reach; then with a group of more rows than a wave holds.
    [(0, 2, 90), (2, 5, 2), (8, 1, 7), (9, 3, 3)],
    [(1, 4, 2), (5, 2, 0), (7, 3, 5), (11, 2, 90)],
    [(0, 3, 4), (3, 2, 61), (6, 40, 3)],
    [(0, 40, 1), (42, 2, 61), (44, 3, 9)],
]


@pytest.mark.parametrize("groups", UNLIKE)
@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
def test_prefixes_of_unlike_lengths(monkeypatch, groups, dtype, kv, scaled):
    page, q_len = 16, 2
    b = groups[-1][0] + groups[-1][1] + 2
    lens = [17 + 5 * i % 60 for i in range(b)]
    for first, count, pages in groups:
        for i in range(first, first + count):
            lens[i] = pages * page + q_len + (7 * i) % 50
    lens[groups[0][0]] -= 40  # padded: it goes over its own row
    q, caches, scales, tables, full, sl = inputs(groups, lens, q_len, 8, 2, 64, page, dtype, kv,
                                                 scaled, seed=b)
    want, bound = ref.attention(q, *caches, *scales, full, sl, everything(q_len),
                                p_step=p_step(dtype, scaled))
    qc, kc, vc, ks, vs, bt, slc = ref.cuda(q, *caches, *scales, tables, sl)

    for size in (1, 4, 7, 30):
        def change(p, shared):
            splits = [_splits(pages, size) for _, pages in shared]
            p.shared_size, even = size, max(splits)
            p.num_items = sum(-(-n * 8 // p.block_rows) * s for (n, _), s in zip(shared, splits))
            p.shared_splits = min(even, -(-(b + sum(n * x for n, x in shared) // size) // b))
            assert p.shared_splits < even

        with monkeypatch.context() as m:
            made = _forge(m, change)
            plan = plan_shared_prefix(groups, b, q_len, 8, 2, 64, page)
            out = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, key_scale=ks,
                                                value_scale=vs)
        assert made and made[-1].shared_size == size
        ref.assert_within(out, want, bound, f"size {size}")


def test_a_long_prefix_of_two_in_a_large_batch():
    """As the plan itself has it: 2 sequences over 16K tokens beside 254 over 64."""
    groups, q_len = [(0, 2, 1024), (2, 254, 4)], 1
    lens = [1024 * 16 + 5, 1024 * 16 + 90] + [64 + 1 + i % 40 for i in range(254)]
    q, (k, v), _, tables, full, sl = inputs(groups, lens, q_len, 8, 2, 128, 16, F16, None, False)
    want, bound = ref.attention(q, k, v, None, None, full, sl, everything(q_len))
    made, need, _ = _lib.plan_shared_prefix(0, tuple(groups), (256, q_len, 8, 2, 128, 16),
                                            _lib.DTYPE_F16, 0, tables.shape[1])
    assert 1 <= made.shared_splits < _splits(1024, made.shared_size)
    assert need < 256 << 20
    args = ref.cuda(q, k, v, tables, sl)
    plan = plan_shared_prefix(groups, 256, q_len, 8, 2, 128, 16)
    ref.assert_within(paged_attention_shared_prefix(*args, plan), want, bound)


# --------------------------------------------------------------------------------------
# Partial rows past 32-bit offsets.
# --------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,kv,scaled", CACHES[:2] + CACHES[4:5])
@pytest.mark.parametrize("count", [2, 10])
def test_partial_rows_past_4_gib(monkeypatch, dtype, kv, scaled, count):
    """Cuts with slots for 100000 splits in all, which nearly all stay empty: own rows on both
    sides of 4 GiB, and past it a group's (of one wave's rows, and in tiles)."""
    page, q_len, hq, hkv, d = 16, 4, 32, 8, 128
    groups, b = [(0, count, 40)], count + 2
    each = 100000 // b
    lens = [640 + 30 + 90 * i for i in range(count)] + [900, 2000]
    q, caches, scales, tables, full, sl = inputs(groups, lens, q_len, hq, hkv, d, page, dtype, kv,
                                                 scaled, seed=count)
    qc, kc, vc, ks, vs, bt, ft, slc = ref.cuda(q, *caches, *scales, tables, full, sl)

    def change(p, shared):
        p.num_splits, p.pages_per_split, p.wg_heads = each, 1, 4

    with monkeypatch.context() as m:
        _forge(m, change)
        plan = plan_shared_prefix(groups, b, q_len, hq, hkv, d, page)
        out = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, key_scale=ks, value_scale=vs)
    assert each * (b - 1) * q_len * hq * d * 4 > 4 << 30
    want, bound = ref.attention(q, *caches, *scales, full, sl, everything(q_len),
                                p_step=p_step(dtype, scaled))
    ref.assert_within(out, want, bound, "shared prefix")
    with monkeypatch.context() as m:
        m.setattr(windowed, "_KNOWN", scaled_cache.Layouts())
        m.setattr(_lib, "plan_windowed", lambda *a: (each, 1, 2))
        out = paged_attention_windowed(qc, kc, vc, ft, slc, 500, sink=9, key_scale=ks, value_scale=vs)
    want, bound = ref.attention(q, *caches, *scales, full, sl,
                                lambda i, n: ref.window_seen(n, q_len, 500, 9))
    ref.assert_within(out, want, bound, "window")


# --------------------------------------------------------------------------------------
# Values that are not finite where every row sees them.
# --------------------------------------------------------------------------------------

INF, NAN = float("inf"), float("nan")


def _put(cache, table, t, head, dim, x):
    """Value x at token t of a table row (e4m3 has no infinities: NaN)."""
    page = cache.shape[1]
    raw = cache.view(torch.uint8) if cache.element_size() == 1 else cache
    raw[int(table[t // page]), t % page, head, dim] = 0x7F if cache.element_size() == 1 else x


@pytest.mark.parametrize("dtype,kv", [(F16, None), (BF16, None), (BF16, E4M3)])
@pytest.mark.parametrize("d,q_len", [(64, 3), (64, 16), (128, 1), (128, 6), (128, 12), (256, 2), (256, 8)])
@pytest.mark.parametrize("sharp", [1, 40])
def test_values_inside_a_window(dtype, kv, d, q_len, sharp):
    """Infinities and NaN on pages that no edge of a window crosses; with large scores too, where
    most probabilities and weights of splits round to 0."""
    hkv, page, window, sink, lens = 2, 16, 2000, 20, [2600, 700, 3000]
    q, (k, v), _, tables, sl = ref.window_inputs(lens, q_len, 4 * hkv, hkv, d, page, dtype, kv, False,
                                                 window, sink, seed=d + q_len)
    q = q * sharp
    for i, t, h, e, x in ((0, 1500, 0, 5, INF), (0, 900, 0, 6, -INF), (0, 2570, 1, 7, NAN),
                          (0, 1000, 1, 9, INF), (0, 2400, 1, 9, -INF), (0, 3, 0, 30, -INF),
                          (1, 33, 1, d - 1, INF), (1, 650, 1, d - 1, INF), (1, 400, 0, 0, -INF)):
        _put(v, tables[i], t, h, e, x)
    want, bound = ref.attention(q, k, v, None, None, tables, sl,
                                lambda i, n: ref.window_seen(n, q_len, window, sink))
    assert want.isnan().any() and (kv or want.isinf().any()) and want[2].isfinite().all()
    qc, kc, vc, bt, slc = ref.cuda(q, k, v, tables, sl)
    for most in (0, 3000):
        out = paged_attention_windowed(qc, kc, vc, bt, slc, window, sink=sink, max_seq_len=most)
        ref.assert_within(out, want, bound, f"max_seq_len {most}")


@pytest.mark.parametrize("dtype,kv", [(F16, None), (BF16, None), (BF16, E4M3)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("count,q_len", [(2, 2), (4, 4), (7, 4), (20, 4), (70, 1)])
@pytest.mark.parametrize("sharp", [1, 40])
def test_values_on_shared_pages(dtype, kv, d, count, q_len, sharp):
    """16 to 320 rows of a kv head: in waves, and in tiles of 128 and 256."""
    hkv, page, shared = 2, 16, 67
    lens = [shared * page + q_len + 11 * i % 300 for i in range(count)]
    lens[1] = 100  # goes over its own row
    q, (k, v), _, tables, full, sl = inputs([(0, count, shared)], lens, q_len, 4 * hkv, hkv, d, page,
                                            dtype, kv, False, seed=count)
    q = q * sharp
    for i, t, h, e, x in ((0, 100, 0, 5, INF), (0, 1000, 0, 6, -INF), (0, 64, 1, 7, NAN),
                          (0, 33, 1, 9, INF), (0, 990, 1, 9, -INF), (0, shared * page - 1, 0, 0, INF),
                          (0, 0, 1, d - 1, -INF), (1, 50, 0, 33, INF),
                          (count - 1, shared * page, 1, 40, INF)):
        _put(v, full[i], t, h, e, x)
    want, bound = ref.attention(q, k, v, None, None, full, sl, everything(q_len),
                                p_step=p_step(dtype, False))
    assert want.isnan().any() and (kv or want.isinf().any()) and want.isfinite().any()
    qc, kc, vc, bt, slc = ref.cuda(q, k, v, tables, sl)
    plan = plan_shared_prefix([(0, count, shared)], count, q_len, 4 * hkv, hkv, d, page)
    ref.assert_within(paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan), want, bound)


@pytest.mark.parametrize("scaled", [E4M3, INT8])
def test_codes_that_are_nan_in_tiles(scaled):
    """Under block scales: NaN codes (e4m3) and NaN scales of a shared page reach all rows that
    share it, in tiles."""
    count, q_len, page, shared, d = 30, 4, 16, 21, 128
    lens = [shared * page + q_len + 7 * i % 90 for i in range(count)]
    q, (k, v), (ks, vs), tables, full, sl = inputs([(0, count, shared)], lens, q_len, 8, 2, d, page,
                                                   BF16, scaled, True, seed=3)
    if scaled is E4M3:
        _put(v, full[0], 200, 1, 9, NAN)
    vs[int(full[0, 3]), 0] = NAN
    want, bound = ref.attention(q, k, v, ks, vs, full, sl, everything(q_len))
    qc, kc, vc, ksc, vsc, bt, slc = ref.cuda(q, k, v, ks, vs, tables, sl)
    plan = plan_shared_prefix([(0, count, shared)], count, q_len, 8, 2, d, page)
    out = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, key_scale=ksc, value_scale=vsc)
    assert want.isnan().any() and want.isfinite().any()
    ref.assert_within(out, want, bound)


# --------------------------------------------------------------------------------------
# Plans and streams.
# --------------------------------------------------------------------------------------

@pytest.mark.parametrize("traced", [False, True])
def test_a_plan_dropped_before_its_call_has_run(traced):
    """A call waits on another stream than its plan was made on, behind a second of other work;
    the plan goes and others are made. The table's memory is nobody's meanwhile."""
    groups, b = [(0, 3, 8), (3, 30, 20)], 33
    lens = [8 * 16 + 5 + i for i in range(3)] + [20 * 16 + 5 + i for i in range(30)]
    q, (k, v), _, tables, full, sl = inputs(groups, lens, 4, 8, 2, 128, 16, F16, None, False)
    args = ref.cuda(q, k, v, tables, sl)

    def call(plan):
        if not traced:
            return paged_attention_shared_prefix(*args, plan)
        return torch.ops.sqa.paged_attention_shared_prefix(
            *args[:3], None, None, *args[3:], None, plan.flat, plan.table, 128 ** -0.5, 1.0, 0)

    want = call(plan_shared_prefix(groups, b, 4, 8, 2, 128, 16)).clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    plan = plan_shared_prefix(groups, b, 4, 8, 2, 128, 16)
    at, size = plan.table.data_ptr(), plan.table.numel()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000_000)
        out = call(plan)
    del plan
    others = [torch.empty(size, dtype=torch.int32, device="cuda") for _ in range(64)]
    assert not side.query()  # the call still waits
    assert all(x.data_ptr() != at for x in others)
    # (Their copies may wait for the other stream: the two can share a queue of the device.)
    del others
    others = [plan_shared_prefix([(0, 33, 1)], b, 4, 8, 2, 128, 16) for _ in range(8)]
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# --------------------------------------------------------------------------------------
# Probabilities of shared pages in tiles.
# --------------------------------------------------------------------------------------

def _heavy(dtype, kv, d, count, keys, seed=0):
    """Queries along dim 0, of 2^0.5 to 2^7.9 against a key of 2: a first key of 0 sets the
    maximum, those of ``keys`` {token: key} carry nearly all of the weight without raising it,
    all others none."""
    q_len, hq, hkv, page, shared = 4, 8, 2, 16, 9
    lens = [shared * page + q_len + i % 60 for i in range(count)]
    q, (k, v), _, tables, full, sl = inputs([(0, count, shared)], lens, q_len, hq, hkv, d, page,
                                            dtype, kv, False, seed)
    size = torch.linspace(0.5, 7.9, q[..., 0].numel()) * d ** 0.5 / 2 * 0.6931471805599453
    q = torch.zeros_like(q)
    q[..., 0] = size.view(q[..., 0].shape).to(dtype)
    k = torch.zeros(k.shape)
    k[..., 0] = -60
    for t, x in {0: 0.0, **keys}.items():
        k[int(full[0, t // page]), t % page, :, 0] = x
    plan = plan_shared_prefix([(0, count, shared)], count, q_len, hq, hkv, d, page)
    return q, k.to(kv or dtype), v, tables, full, sl, plan


TILES = [(d, count) for d in (64, 128, 256) for count in (7, 33)]  # 112 and 528 rows of a kv head


@pytest.mark.parametrize("d,count", TILES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_probabilities_over_e4m3_have_11_bits(dtype, d, count):
    """Two keys share a row's weight, their values opposite."""
    q, k, v, tables, full, sl, plan = _heavy(dtype, E4M3, d, count, {40: 2.0, 41: 1.875})
    raw = v.view(torch.uint8)
    raw[int(full[0, 2]), 9] = raw[int(full[0, 2]), 8] ^ 0x80
    want, bound = ref.attention(q, k, v, None, None, full, sl, everything(4), p_step=2.0 ** -11)
    out = paged_attention_shared_prefix(*ref.cuda(q, k, v, tables, sl), plan)
    ref.assert_within(out, want, bound)


@pytest.mark.parametrize("d,count", TILES)
@pytest.mark.parametrize("dtype,kv", [(F16, None), (BF16, None), (F16, E4M3), (BF16, E4M3)])
def test_weights_of_a_row_add_up_to_one(dtype, kv, d, count):
    """Where all tokens have one value, so has every row, to the bit: the rounding of a heavy
    probability is in its row's sum as in the product."""
    q, k, v, tables, full, sl, plan = _heavy(dtype, kv, d, count, {40: 2.0})
    # (A weight off by more than 2^-9 shows in values just below a power of two, where the steps of
    # the type are smallest beside the value.)
    value = torch.tensor([1.875, -3.75]).repeat(d // 2)
    v = torch.zeros(v.shape).add(value).to(v.dtype)
    out = paged_attention_shared_prefix(*ref.cuda(q, k, v, tables, sl), plan)
    assert torch.equal(out.float().cpu(), value.expand(q.shape))


# --------------------------------------------------------------------------------------
# All of it at once.
# --------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,splits,items", [(1, 1, 0), (4, 3, 0), (2, 40, 0), (1, 0, 1), (2, 0, 5),
                                                (4, 0, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_values_at_every_cut_of_a_window(monkeypatch, dtype, heads, splits, items):
    """Infinities in pieces of items that cross sequence ends, and in parts of several waves."""
    lens, q_len, hq, hkv, d, page, window, sink = [700, 0, 33, 1500, 64, 900], 3, 12, 3, 64, 16, 600, 9
    q, (k, v), _, tables, sl = ref.window_inputs(lens, q_len, hq, hkv, d, page, dtype, None, False,
                                                 window, sink, seed=items)
    for i, n in enumerate(lens):
        for t, h, e, x in ((n // 2 + 200, 0, 1, INF), (n - 40, 2, 5, -INF), (n - 300, 1, 8, INF),
                           (n - 200, 1, 8, -INF), (2, 2, 30, INF)):
            if 0 <= t < n and (t < sink or t >= n - q_len + 1 - window):
                _put(v, tables[i], t, h, e, x)
    monkeypatch.setattr(windowed, "_KNOWN", scaled_cache.Layouts())
    monkeypatch.setattr(_lib, "plan_windowed", lambda *a: (
        splits or items + len(lens), int(splits > 0), heads))
    out = paged_attention_windowed(*ref.cuda(q * 20, k, v, tables, sl), window, sink=sink)
    want, bound = ref.attention(q * 20, k, v, None, None, tables, sl,
                                lambda i, n: ref.window_seen(n, q_len, window, sink))
    assert want.isinf().any() and want.isnan().any()
    ref.assert_within(out, want, bound)


@pytest.mark.parametrize("seed", range(40))
def test_drawn_batches(monkeypatch, seed):
    """Drawn groups of unlike lengths, padded and short sequences, split sizes, values that are
    not finite where somebody sees them."""
    g = torch.Generator().manual_seed(5000 + seed)

    def draw(n):
        return int(torch.randint(n, (1,), generator=g))

    dtype, kv, scaled = CACHES[draw(len(CACHES))]
    d, page, hkv, group = (64, 128, 256)[draw(3)], (16, 16, 64)[draw(3)], 1 + draw(4), 1 + draw(8)
    q_len = 1 + draw(max(1, min(8, (32 if d == 256 else 64) // group)))
    groups, lens = [], []
    for _ in range(1 + draw(5)):
        lens += [draw(150) for _ in range(draw(3))]
        count, pages = 1 + draw((4, 30)[draw(2)]), draw((5, 60)[draw(2)] * 16 // page + 1)
        groups.append((len(lens), count, pages))
        lens += [pages * page + q_len + draw(200) if draw(6) else draw(pages * page + 40)
                 for _ in range(count)]
    b = len(lens)
    if max(lens) == 0:
        lens[0] = 5
    q, caches, scales, tables, full, sl = inputs(groups, lens, q_len, hkv * group, hkv, d, page, dtype,
                                                 kv, scaled, seed)
    if not scaled and draw(2):
        for _ in range(6):
            i = draw(b)
            if lens[i]:
                _put(caches[1], full[i], draw(lens[i]), draw(hkv), draw(d), (INF, -INF, NAN)[draw(3)])
    size = 1 + draw(40)

    def change(p, shared):
        splits = [_splits(pages, size) for _, pages in shared]
        if not p.num_items:
            return
        rows = q_len * group
        p.shared_size, even = size, max(splits)
        p.num_items = sum(-(-n * rows // p.block_rows) * s for (n, _), s in zip(shared, splits))
        p.shared_splits = min(even, -(-(b + sum(n * x for n, x in shared) // size) // b))

    qc, kc, vc, ks, vs, bt, slc = ref.cuda(q, *caches, *scales, tables, sl)
    want, bound = ref.attention(q, *caches, *scales, full, sl, everything(q_len),
                                p_step=p_step(dtype, scaled))
    for forged in (False, True):
        with monkeypatch.context() as m:
            if forged:
                _forge(m, change)
            plan = plan_shared_prefix(groups, b, q_len, hkv * group, hkv, d, page)
            out = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, key_scale=ks,
                                                value_scale=vs)
        ref.assert_within(out, want, bound, f"forged {forged}")
