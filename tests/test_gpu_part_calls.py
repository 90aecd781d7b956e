"""How attention over a window and over a shared prefix is called on the GPU: beside the other
operators of a decoding step, captured in graphs, on several streams and threads, traced, over
large pools, with every way to cut a batch."""

import ctypes
import threading

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd import _lib, scaled_cache, windowed  # noqa: E402
from small_q_attention_amd.masks import pack_draft_mask  # noqa: E402
from small_q_attention_amd.shared_prefix import (paged_attention_shared_prefix,  # noqa: E402
                                                 plan_shared_prefix)
from small_q_attention_amd.windowed import paged_attention_windowed  # noqa: E402
from tests import _cache_reference, _part_reference as ref  # noqa: E402
from tests._part_reference import BF16, E4M3, F16, INT8  # noqa: E402
from tests.test_gpu_shared_prefix import inputs as prefix_inputs, p_step  # noqa: E402

pytestmark = pytest.mark.gpu

CACHES = [(F16, None, False), (BF16, None, False), (F16, E4M3, False), (BF16, E4M3, False),
          (F16, E4M3, True), (BF16, INT8, True)]
GROUPS, PAGE, Q, HQ, HKV, D = [(0, 4, 12), (5, 2, 3)], 16, 4, 8, 2, 128
LENS = [12 * 16 + 40, 12 * 16 + 4, 12 * 16 + 300, 500, 90, 3 * 16 + 9, 700]
WINDOW, SINK = 150, 6


def _cpu_state(seed, lens=LENS, dtype=F16, kv=INT8, scaled=True):
    """What a step takes, sequences of one group on the same shared pages; a pool and tables
    of one size whatever the lengths."""
    g = torch.Generator().manual_seed(seed)
    b, width = len(lens), 48
    pool = b * width
    tables = torch.randperm(pool, generator=g).to(torch.int32).view(b, width)
    for first, count, pages in GROUPS:
        tables[first:first + count, :pages] = tables[first, :pages]
    q = torch.randn(b, Q, HQ, D, generator=g).to(dtype)
    caches, scales = zip(*(ref.cache(pool, PAGE, HKV, D, dtype, kv, scaled, g) for _ in range(2)))
    key, value = (torch.randn(b, Q, HKV, D, generator=g).to(dtype) for _ in range(2))
    names = ("query", "k", "v", "ks", "vs", "tables", "lens", "key", "value")
    return dict(zip(names, (q, *caches, *scales, tables, torch.tensor(lens, dtype=torch.int32),
                            key, value)))


def _state(*a, **kw):
    s = _cpu_state(*a, **kw)
    return dict(zip(s, ref.cuda(*s.values())))


def _plan():
    return plan_shared_prefix(GROUPS, len(LENS), Q, HQ, HKV, D, PAGE)


def _step(s, plan, **kw):
    """One pass of a decoding loop: the step's keys and values are quantised into the cache,
    one layer reads a window of it, another all of it."""
    if s["ks"] is not None:
        scaled_cache.append_scaled_kv(s["key"], s["value"], s["k"], s["v"], s["ks"], s["vs"],
                                      s["tables"], s["lens"])
    args = [s[n] for n in ("query", "k", "v", "tables", "lens")]
    scales = dict(key_scale=s["ks"], value_scale=s["vs"], **kw)
    local = paged_attention_windowed(*args, WINDOW, sink=SINK, **scales)
    return [local, paged_attention_shared_prefix(local, *args[1:], plan, **scales)]


def _load(s, t):
    for n in s:
        if s[n] is not None:
            s[n].copy_(t[n])


@pytest.mark.parametrize("dtype,kv", [(F16, E4M3), (F16, INT8), (BF16, INT8)])
def test_a_step_beside_the_quantising_append(dtype, kv):
    """Against the plain statement of all three in turn; the second attention is asked with
    the first one's result."""
    c = _cpu_state(1, dtype=dtype, kv=kv)
    local, whole = (x.cpu() for x in _step(_state(1, dtype=dtype, kv=kv), _plan()))
    caches, scales = [c["k"], c["v"]], [c["ks"], c["vs"]]
    # (Shared pages are whole before any sequence's new tokens: appends leave them alone.)
    _cache_reference.append(c["key"], c["value"], caches, scales, c["tables"], c["lens"])
    s = _state(1, dtype=dtype, kv=kv)
    scaled_cache.append_scaled_kv(s["key"], s["value"], s["k"], s["v"], s["ks"], s["vs"],
                                  s["tables"], s["lens"])
    for a, w in zip((s["ks"], s["vs"]), scales):
        assert torch.equal(a.cpu(), w)
    caches = [x.cpu() for x in (s["k"], s["v"])]  # (codes on a border may round either way)
    for q, out, seen in ((c["query"], local, lambda i, n: ref.window_seen(n, Q, WINDOW, SINK)),
                         (local, whole, lambda i, n: ref.window_seen(n, Q, 1 << 30, 0))):
        want, bound = ref.attention(q, *caches, *scales, c["tables"], c["lens"], seen)
        ref.assert_within(out, want, bound)


@pytest.mark.parametrize("dtype,kv,scaled", [(F16, None, False), (BF16, None, False),
                                             (F16, E4M3, False), (BF16, INT8, True)])
def test_a_step_captured_in_a_graph(dtype, kv, scaled):
    """Replays with other data, lengths among it, give the eager calls' bits, with eager calls
    and synchronisations between them."""
    how = dict(dtype=dtype, kv=kv, scaled=scaled)
    s, plan = _state(1, **how), _plan()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(s, plan)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(s, plan)
    b = len(LENS)
    for seed, lens in ((2, LENS), (3, [768] * b), (4, [0, 5, 300, 16, 700, 2, 52]), (5, [0] * b),
                       (6, [n + 13 for n in LENS])):
        want = _step(_state(seed, lens, **how), plan)
        _load(s, _state(seed, lens, **how))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want)), (seed, lens)
        assert lens != [0] * b or not any(x.any() for x in got)


def test_two_graphs_replayed_at_once():
    """Each graph's workspaces are its own."""
    plan = _plan()
    states, graphs, outs = [_state(7), _state(8)], [], []
    for s in states:
        _step(s, plan)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(s, plan))
        graphs.append(g)
    want = [_step(_state(i), plan) for i in (7, 8)]
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, i in zip(states, (7, 8)):
            _load(s, _state(i))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_calls_on_several_streams():
    plan = _plan()
    want = [_step(_state(10 + i), plan) for i in range(4)]
    states = [_state(10 + i) for i in range(4)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in states], []
    for s, st in zip(states, streams):
        with torch.cuda.stream(st):
            outs.append(_step(s, plan))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_host_threads_on_one_stream():
    """Two threads' calls under one plan, their kernels launched between each other's."""
    states, plan = [_state(20 + i, kv=None, scaled=False) for i in range(2)], _plan()
    want = [_step(s, plan) for s in states]
    torch.cuda.synchronize()
    got, errors, start = [[], []], [], threading.Barrier(2)

    def worker(i):
        try:
            start.wait()
            for _ in range(20):
                got[i].append(_step(states[i], plan))
        except Exception as exc:  # reported by the main thread
            errors.append(repr(exc))

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 20
        assert all(torch.equal(a, w) for o in got[i] for a, w in zip(o, want[i]))


@pytest.mark.parametrize("kv,scaled", [(None, False), (INT8, True)])
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_traced_calls(kv, scaled, backend):
    """torch.compile (fullgraph) runs the custom ops; the bits are the eager calls'."""
    plan = _plan()
    names = ("query", "k", "v", "tables", "lens", "ks", "vs")

    def step(query, k, v, tables, lens, ks, vs):
        scales = dict(key_scale=ks, value_scale=vs)
        a = paged_attention_windowed(query, k, v, tables, lens, WINDOW, sink=SINK, **scales)
        return a + 1, paged_attention_shared_prefix(a, k, v, tables, lens, plan, **scales) * 2

    s = _state(30, kv=kv, scaled=scaled)
    args = [s[n] for n in names]
    want = step(*args)
    got = torch.compile(step, backend=backend, fullgraph=True)(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_on_the_device():
    s, plan = _state(31, kv=None, scaled=False), _plan()
    args = [s[n] for n in ("query", "k", "v", "tables", "lens")]
    odd = torch.empty(s["query"].numel() + 1, dtype=F16, device="cuda")[1:].view(s["query"].shape)
    for call in (lambda q, *a, **kw: paged_attention_windowed(q, *a, 5, **kw),
                 lambda q, *a, **kw: paged_attention_shared_prefix(q, *a, plan, **kw)):
        with pytest.raises(ValueError, match="16-byte"):
            call(odd, *args[1:])
        with pytest.raises(ValueError, match="must not be query"):
            call(*args, out=s["query"])
        with pytest.raises(ValueError, match="out must be"):
            call(*args, out=s["query"].float())
        with pytest.raises(ValueError, match="GPU"):
            call(*args[:4], s["lens"].cpu())
    with pytest.raises(ValueError, match="made for"):
        paged_attention_shared_prefix(s["query"][:, :2].contiguous(), *args[1:], plan)
    with pytest.raises(ValueError, match="shares 12 pages"):
        paged_attention_shared_prefix(*args[:3], s["tables"][:, :11].contiguous(), s["lens"], plan)


# --------------------------------------------------------------------------------------
# Large pools.
# --------------------------------------------------------------------------------------

def test_pools_past_32_bit_offsets():
    """Pages past 4 GiB of a pool, among them shared ones: in waves and in tiles."""
    page, hkv, d, q_len, hq = 64, 8, 128, 4, 16
    pages = (5 << 30) // (page * hkv * d * 2)
    k, v = (torch.zeros(pages, page, hkv, d, dtype=F16, device="cuda") for _ in range(2))
    for groups, b in (([(0, 3, 4)], 3), ([(0, 12, 4)], 12)):
        lens = [4 * page + 7 + 9 * i for i in range(b)]
        q, (ks, vs), _, _, full, sl = prefix_inputs(groups, lens, q_len, hq, hkv, d, page, F16, None,
                                                    False, seed=b)
        n = ks.shape[0]
        at = torch.cat([torch.arange(n // 2), pages - 1 - torch.arange(n - n // 2)])
        k[at.cuda()], v[at.cuda()] = ks.cuda(), vs.cuda()
        assert (full[:, :4] >= n // 2).any()
        tables = torch.where(full < 0, -1, at[full.clamp(min=0).long()]).to(torch.int32)
        args = ref.cuda(q) + [k, v] + ref.cuda(tables, sl)
        plan = plan_shared_prefix(groups, b, q_len, hq, hkv, d, page)
        want, bound = ref.attention(q, ks, vs, None, None, full, sl,
                                    lambda i, n: ref.window_seen(n, q_len, 1 << 30, 0))
        ref.assert_within(paged_attention_shared_prefix(*args, plan), want, bound)
        want, bound = ref.attention(q, ks, vs, None, None, full, sl,
                                    lambda i, n: ref.window_seen(n, q_len, 90, 70))
        ref.assert_within(paged_attention_windowed(*args, 90, sink=70), want, bound)


def test_scales_of_heads_past_32_bit_offsets():
    """Scales whose heads lie 1 GiB apart."""
    hkv, d, page, far = 8, 64, 16, 1 << 28
    store = [torch.empty(hkv * far, device="cuda") for _ in range(2)]
    for groups, b in (([(0, 3, 4)], 3), ([(0, 40, 4)], 40)):
        lens = [4 * page + 3 + i % 17 for i in range(b)]
        q, caches, scales, tables, full, sl = prefix_inputs(groups, lens, 2, 16, hkv, d, page, F16,
                                                            INT8, True, seed=b)
        ks, vs = (x.as_strided(s.shape, (1, far)) for x, s in zip(store, scales))
        ks.copy_(scales[0])
        vs.copy_(scales[1])
        args = ref.cuda(q, *caches, full, sl)
        plan = plan_shared_prefix(groups, b, 2, 16, hkv, d, page)
        want, bound = ref.attention(q, *caches, *scales, full, sl,
                                    lambda i, n: ref.window_seen(n, 2, 1 << 30, 0))
        ref.assert_within(paged_attention_shared_prefix(*args, plan, key_scale=ks, value_scale=vs),
                          want, bound)
        want, bound = ref.attention(q, *caches, *scales, full, sl,
                                    lambda i, n: ref.window_seen(n, 2, 20, 3))
        ref.assert_within(paged_attention_windowed(*args, 20, sink=3, key_scale=ks, value_scale=vs),
                          want, bound)


# --------------------------------------------------------------------------------------
# Cuts that the plans may choose, whatever the device's size.
# --------------------------------------------------------------------------------------

CUTS = [(heads, splits, items) for heads in (1, 2, 4)
        for splits, items in ((1, 0), (3, 0), (40, 0), (0, 1), (0, 5), (0, 64))]


@pytest.mark.parametrize("heads,splits,items", CUTS)
@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
def test_every_cut_of_a_window(monkeypatch, dtype, kv, scaled, heads, splits, items):
    """Three kv heads (a workgroup of two or four has one too many), empty sequences first,
    last and between, more than a wave's lanes of them."""
    lens = [0, 0] + [(61 * i) % 300 if i % 5 else 0 for i in range(70)] + [1200, 0, 0, 30, 0]
    q, caches, scales, tables, sl = ref.window_inputs(lens, 2, 6, 3, 64, 16, dtype, kv, scaled, 120,
                                                      20, seed=items)
    monkeypatch.setattr(windowed, "_KNOWN", scaled_cache.Layouts())
    monkeypatch.setattr(_lib, "plan_windowed", lambda *a: (
        splits or items + len(lens), int(splits > 0), heads))
    qc, kc, vc, ks, vs, bt, slc = ref.cuda(q, *caches, *scales, tables, sl)
    out = paged_attention_windowed(qc, kc, vc, bt, slc, 120, sink=20, key_scale=ks, value_scale=vs)
    want, bound = ref.attention(q, *caches, *scales, tables, sl,
                                lambda i, n: ref.window_seen(n, 2, 120, 20))
    ref.assert_within(out, want, bound)


def _recut(monkeypatch, heads, splits, items, size):
    """Shared-prefix plans of this cut in place of the model's."""
    real = _lib.plan_shared_prefix

    def forged(device, groups, shape, kv, most, width):
        made, _, table = real(device, groups, shape, kv, most, width)
        p = _lib.SharedPlan()
        ctypes.memmove(ctypes.byref(p), ctypes.byref(made), ctypes.sizeof(made))
        p.wg_heads, p.pages_per_split = heads, int(splits > 0)
        p.num_splits = splits or items + p.batch
        p.shared_size, p.num_items, p.shared_splits = size, 0, 0
        rows = p.q_len * (p.num_query_heads // p.num_kv_heads)
        for _, count, pages in groups:
            pages *= (p.page_size // 16) * (count > 1)
            if pages:
                each = -(-pages // -(-pages // size))
                p.shared_splits = max(p.shared_splits, -(-pages // each))
                p.num_items += -(-count * rows // p.block_rows) * -(-pages // each)
        return p, int(_lib.load().sqa_shared_workspace_bytes(ctypes.byref(p))), table

    monkeypatch.setattr(_lib, "plan_shared_prefix", forged)


@pytest.mark.parametrize("heads,splits,items", CUTS)
@pytest.mark.parametrize("rows", [16, 64, 256])
def test_every_cut_of_a_batch_that_shares(monkeypatch, rows, heads, splits, items):
    """Blocks of a wave and of eight waves; sequences of no group, short ones and empty ones
    between the groups."""
    monkeypatch.setattr(windowed, "_KNOWN", scaled_cache.Layouts())
    count = rows // 4
    lens = [0, 100] + [160 + 4 + (37 * i) % 150 for i in range(count)] + [0, 30, 900, 160, 90, 5]
    groups = [(2, count, 10), (count + 4, 2, 2)]
    q, caches, _, tables, full, sl = prefix_inputs(groups, lens, 2, 6, 3, 64, 16, F16, None, False,
                                                   seed=rows)
    want, bound = ref.attention(q, *caches, None, None, full, sl,
                                lambda i, n: ref.window_seen(n, 2, 1 << 30, 0))
    args = ref.cuda(q, *caches, tables, sl)
    for size in (10, 4, 1):
        _recut(monkeypatch, heads, splits, items, size)
        plan = plan_shared_prefix(groups, len(lens), 2, 6, 3, 64, 16)
        ref.assert_within(paged_attention_shared_prefix(*args, plan), want, bound, f"size {size}")


@pytest.mark.parametrize("dtype,kv,scaled", CACHES)
@pytest.mark.parametrize("wide", [2, 70])
def test_more_groups_than_a_wave_has_lanes(dtype, kv, scaled, wide):
    """150 groups, one of `wide` sequences (140 rows: in tiles) among them."""
    groups, lens, at = [], [], 0
    for i in range(150):
        count = wide if i == 97 else 1 + i % 3
        pages = i % 4
        groups.append((at, count, pages))
        lens += [pages * 16 + 2 + (5 * (at + j)) % 40 for j in range(count)]
        at += count
    q, caches, scales, tables, full, sl = prefix_inputs(groups, lens, 2, 2, 2, 64, 16, dtype, kv,
                                                        scaled, seed=wide)
    want, bound = ref.attention(q, *caches, *scales, full, sl,
                                lambda i, n: ref.window_seen(n, 2, 1 << 30, 0),
                                p_step=p_step(dtype, scaled))
    qc, kc, vc, ks, vs, bt, slc = ref.cuda(q, *caches, *scales, tables, sl)
    plan = plan_shared_prefix(groups, len(lens), 2, 2, 2, 64, 16)
    out = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, key_scale=ks, value_scale=vs)
    ref.assert_within(out, want, bound)


@pytest.mark.parametrize("kv", [E4M3, INT8])
@pytest.mark.parametrize("d,count", [(64, 2), (128, 9), (128, 70), (256, 40)])
def test_scales_of_pages_nobody_has(kv, d, count):
    """Loads past a split's last page take place 0's scale along: NaN here."""
    lens = [5 * 16 + 3 + i % 40 for i in range(count)]
    q, caches, scales, _, full, sl = prefix_inputs([(0, count, 5)], lens, 2, 8, 2, d, 16, F16, kv,
                                                   True, seed=d)
    caches = [torch.cat([c[:1].view(torch.uint8), c.view(torch.uint8)]).view(kv) for c in caches]
    scales = [torch.cat([torch.full((1, 2), float("nan")), s]) for s in scales]
    full = torch.where(full < 0, 0, full + 1)
    for c in caches:
        ref.spoil(c, [0])
    qc, kc, vc, ks, vs, bt, slc = ref.cuda(q, *caches, *scales, full, sl)
    plan = plan_shared_prefix([(0, count, 5)], count, 2, 8, 2, d, 16)
    want, bound = ref.attention(q, *caches, *scales, full, sl,
                                lambda i, n: ref.window_seen(n, 2, 1 << 30, 0))
    ref.assert_within(paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, key_scale=ks,
                                                    value_scale=vs), want, bound)
    want, bound = ref.attention(q, *caches, *scales, full, sl,
                                lambda i, n: ref.window_seen(n, 2, 20, 2))
    ref.assert_within(paged_attention_windowed(qc, kc, vc, bt, slc, 20, sink=2, key_scale=ks,
                                               value_scale=vs), want, bound)


@pytest.mark.parametrize("seed", range(48))
def test_drawn_calls(seed):
    """Both operators over drawn shapes, lengths, types, layouts and trees."""
    g = torch.Generator().manual_seed(1000 + seed)

    def pick(*xs):
        return xs[int(torch.randint(len(xs), (1,), generator=g))]

    dtype, kv, scaled = pick(*CACHES)
    d, page, hkv, group = pick(64, 128, 256), pick(16, 16, 32, 128), pick(1, 2, 3, 8), pick(1, 2, 4, 7)
    q_len = 1 + int(torch.randint((32 if d == 256 else 64) // group, (1,), generator=g)) \
        if pick(0, 1) else pick(1, 2, 4)
    pages, count = pick(1, 3, 17), pick(2, 6, 24)
    b = count + pick(0, 1, 3)
    lens = [max(0, int(torch.randint(-20, pages * page + 300, (1,), generator=g)))
            for _ in range(b - count)]
    lens += [pages * page + q_len + int(torch.randint(0, 200, (1,), generator=g))
             for _ in range(count)]
    groups = [(b - count, count, pages)]
    tree = ref.trees(b, q_len, seed) if pick(0, 1) else None
    hq = hkv * group
    q, caches, scales, tables, full, sl = prefix_inputs(groups, lens, q_len, hq, hkv, d, page, dtype,
                                                        kv, scaled, seed)
    mask = None if tree is None else pack_draft_mask(tree).cuda()
    qc, kc, vc, ks, vs, bt, ft, slc = ref.cuda(q, *caches, *scales, tables, full, sl)
    plan = plan_shared_prefix(groups, b, q_len, hq, hkv, d, page)
    out = paged_attention_shared_prefix(qc, kc, vc, bt, slc, plan, key_scale=ks, value_scale=vs,
                                        mask=mask)
    of = lambda window, sink: lambda i, n: ref.window_seen(  # noqa: E731
        n, q_len, window, sink, None if tree is None else tree[i])
    want, bound = ref.attention(q, *caches, *scales, full, sl, of(1 << 30, 0),
                                p_step=p_step(dtype, scaled))
    ref.assert_within(out, want, bound, "shared prefix")
    window, sink = pick(1, 30, 129, 5000), pick(0, 3, 40)
    out = paged_attention_windowed(qc, kc, vc, ft, slc, window, sink=sink, key_scale=ks,
                                   value_scale=vs, mask=mask)
    want, bound = ref.attention(q, *caches, *scales, full, sl, of(window, sink))
    ref.assert_within(out, want, bound, "window")


def test_lengths_up_to_the_largest():
    """Lengths past the table are held to it: the largest there is acts as any other."""
    tops = [2**31 - 1, 2**31 - 15, 2**31 - 16, 2**31 - 17] + [2**31 - 1] * 3
    plan = _plan()
    # (Far enough past for a window, which ends at the length, to lie behind the table.)
    past = _step(_state(40, [48 * 16 + 1000] * 7, kv=None, scaled=False), plan)
    top = _step(_state(40, tops, kv=None, scaled=False), plan)
    for a, w in zip(top, past):
        assert torch.equal(a, w) and a.any()


def test_a_wide_window_and_many_first_tokens_are_held_to_the_sequence():
    s = _state(41, kv=None, scaled=False)
    args = [s[n] for n in ("query", "k", "v", "tables", "lens")]
    want = paged_attention_windowed(*args, 48 * 16)
    for window, sink in ((2**31 - 1, 0), (2**40, 0), (2**31 - 1, 2**31 - 1), (1, 2**31 - 1)):
        out = paged_attention_windowed(*args, window, sink=sink)
        assert (out - want).abs().max() < 2e-3
