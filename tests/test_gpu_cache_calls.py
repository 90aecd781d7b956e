"""How the operators around the paged cache are called on the GPU: captured in graphs, on
several streams, traced, through the FlashInfer-shaped entries, over large pools."""

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd import decode_api, eviction, scaled_cache  # noqa: E402
from small_q_attention_amd.masks import pack_draft_mask  # noqa: E402
from tests import _cache_reference as ref  # noqa: E402
from tests.test_gpu_scaled_cache import _cuda, _inputs, _trees  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3, INT8, F16, BF16 = torch.float8_e4m3fn, torch.int8, torch.float16, torch.bfloat16


def _state(seed, lens=(300, 77, 513), q_len=4, dtype=F16, kv=E4M3):
    """Everything a step of all four operators takes, on the GPU."""
    hq, hkv, d, page, budget = 8, 2, 128, 16, 48
    q, caches, scales, tables, sl = _inputs(list(lens), q_len, hq, hkv, d, page, dtype, kv, seed,
                                            width=36)
    # A pool of one size whatever the lengths.
    spare = 120 - caches[0].shape[0]
    caches = [torch.cat([c.view(torch.uint8), torch.zeros(spare, page, hkv, d, dtype=torch.uint8)])
              .view(kv) for c in caches]
    scales = [torch.cat([s, torch.ones(spare, hkv)]) for s in scales]
    for c, s in zip(caches, scales):  # every slot holds something
        c.view(torch.uint8)[(c.view(torch.uint8) & 0x7F) == 0x7F] = 0x30
        s.nan_to_num_(nan=0.01)
    g = torch.Generator().manual_seed(seed + 1)
    key, value = (torch.randn(len(lens), q_len, hkv, d, generator=g).to(dtype) for _ in range(2))
    into = [torch.zeros(3 * len(lens), page, hkv, d, dtype=torch.uint8).view(kv) for _ in range(2)]
    new_tables = torch.randperm(3 * len(lens), generator=g).view(len(lens), 3).to(torch.int32)
    # Entries past a sequence's pages: any page, never read.
    tables = torch.where(tables < 0, 0, tables)
    names = ("query", "k", "v", "ks", "vs", "tables", "lens", "key", "value", "into_k", "into_v",
             "into_ks", "into_vs", "new_tables", "weights")
    values = (q, *caches, *scales, tables, sl, key, value, *into,
              torch.zeros(3 * len(lens), hkv), torch.zeros(3 * len(lens), hkv), new_tables,
              torch.rand(len(lens), hkv, 36 * page, generator=g))
    s = dict(zip(names, _cuda(*values)))
    s["budget"] = budget
    return s


def _step(s):
    """One pass of a decoding loop, everything it returns or writes."""
    scaled_cache.append_scaled_kv(s["key"], s["value"], s["k"], s["v"], s["ks"], s["vs"],
                                  s["tables"], s["lens"])
    out = scaled_cache.paged_attention_scaled(s["query"], s["k"], s["v"], s["ks"], s["vs"],
                                              s["tables"], s["lens"])
    eviction.accumulate_attention_weights(s["query"], s["k"], s["tables"], s["lens"], s["weights"],
                                          key_scale=s["ks"])
    lens, weights, kept = eviction.evict_by_weight(
        s["weights"], s["k"], s["v"], s["tables"], s["lens"], s["new_tables"], s["budget"], sink=2,
        recent=5, key_scale=s["ks"], value_scale=s["vs"],
        into=(s["into_k"], s["into_v"], s["into_ks"], s["into_vs"]))
    return [out, lens, weights, kept, s["k"], s["v"], s["ks"], s["vs"], s["weights"], s["into_k"],
            s["into_v"], s["into_ks"], s["into_vs"]]


def _bits(xs):
    return [x.view(torch.uint8).clone() if x.element_size() == 1 else x.clone() for x in xs]


def _equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(_bits(a), _bits(b)))


def _load(s, t):
    """New data into the state's own buffers."""
    for k, v in t.items():
        if torch.is_tensor(v):
            (s[k].view(torch.uint8) if v.element_size() == 1 else s[k]).copy_(
                v.view(torch.uint8) if v.element_size() == 1 else v)


@pytest.mark.parametrize("dtype,kv", [(F16, E4M3), (BF16, INT8)])
def test_a_step_captured_in_a_graph(dtype, kv):
    """Replays with other data, lengths among it, give the eager calls' bits, with eager
    calls and synchronisations between them."""
    s = _state(1, dtype=dtype, kv=kv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(s)
    for seed, lens in ((2, (300, 77, 513)), (3, (64, 400, 5)), (4, (0, 576, 48)), (5, (3, 17, 16))):
        new = _state(seed, lens, dtype=dtype, kv=kv)
        want = _bits(_step(_state(seed, lens, dtype=dtype, kv=kv)))
        _load(s, new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(_bits(got), want)), (seed, lens)
        _step(new)


def test_two_graphs_replayed_in_turn():
    """Each graph's workspaces are its own."""
    states = [_state(6, (500, 33, 70)), _state(7, (20, 570, 111))]
    graphs, outs = [], []
    for s in states:
        _step(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(s))
        graphs.append(g)
    fresh = [(6, (500, 33, 70)), (7, (20, 570, 111))]
    want = [_bits(_step(_state(*f))) for f in fresh]
    for s, f in zip(states, fresh):
        _load(s, _state(*f))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for g, st in zip(graphs, streams):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(_bits(o), w))


def test_calls_on_several_streams():
    """Calls on other streams than the tensors' own, in turn and at once, give the bits of
    the calls made alone."""
    want = [_bits(_step(_state(10 + i))) for i in range(4)]
    states = [_state(10 + i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    outs = []
    for s, st in zip(states, streams):
        with torch.cuda.stream(st):
            outs.append(_step(s))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(_bits(o), w))


def test_attention_into_a_callers_workspace():
    s = _state(20)
    args = [s[k] for k in ("query", "k", "v", "ks", "vs", "tables", "lens")]
    want = scaled_cache.paged_attention_scaled(*args)
    ws = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(want)
    got = scaled_cache.paged_attention_scaled(*args, out=out, workspace_buffer=ws)
    assert got is out and torch.equal(out, want)
    with pytest.raises(ValueError, match="workspace"):
        scaled_cache.paged_attention_scaled(*args, workspace_buffer=ws[:64])
    with pytest.raises(ValueError, match="16-byte"):
        scaled_cache.paged_attention_scaled(
            torch.empty(s["query"].numel() + 1, dtype=F16, device="cuda")[1:]
            .view(s["query"].shape), *args[1:])


@pytest.mark.parametrize("kv", [E4M3, INT8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_the_flashinfer_shaped_entries(layout, kv):
    b, q_len, hq, hkv, d, page = 3, 4, 8, 2, 128, 16
    q, caches, scales, tables, sl = _inputs([300, 77, 513], q_len, hq, hkv, d, page, F16, kv, 30)
    trees = _trees(b, q_len, 31, (1,))
    pool = torch.stack([c.view(torch.uint8) for c in caches], 1)
    if layout == "HND":
        pool = pool.transpose(2, 3).contiguous()
    pool = pool.cuda().view(kv)
    qc, ks, vs, bt, slc = _cuda(q.view(b * q_len, hq, d), *scales, tables, sl)
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl, trees, scale=0.1, out_scale=2.0)
    out = torch.empty_like(qc)
    for entry in (decode_api.xqa_batch_decode_with_kv_cache,
                  decode_api.trtllm_batch_decode_with_kv_cache):
        got = entry(qc, pool, ws, bt, slc, 513, 0.1, 2.0, kv_layout=layout, q_len_per_req=q_len,
                    mask=pack_draft_mask(trees).cuda(), kv_block_scales=(ks, vs), out=out)
        assert got is out
        ref.assert_within(got.view(q.shape), want, bound)
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl)
    used = [-(-n // page) for n in (300, 77, 513)]
    indptr = torch.tensor([0, used[0], sum(used[:2]), sum(used)], dtype=torch.int32).cuda()
    indices = torch.cat([tables[i, :n] for i, n in enumerate(used)]).cuda()
    last = torch.tensor([(n - 1) % page + 1 for n in (300, 77, 513)], dtype=torch.int32).cuda()
    w = decode_api.BatchDecodeWithPagedKVCacheWrapper(ws, layout)
    w.plan(indptr, indices, last, hq, hkv, d, page, q_data_type=F16, kv_data_type=kv,
           q_len_per_req=q_len)
    ref.assert_within(w.run(qc, pool, kv_block_scales=(ks, vs)).view(q.shape), want, bound)
    if kv is INT8:
        with pytest.raises(ValueError):
            w.run(qc, pool)
    with pytest.raises(ValueError):
        w.run(qc, pool, kv_block_scales=(ks,))


def test_traced_calls():
    """torch.compile (fullgraph) runs the custom ops; the bits are the eager calls'."""
    def step(query, key, value, k, v, ks, vs, tables, lens, weights, new_tables, *into):
        scaled_cache.append_scaled_kv(key, value, k, v, ks, vs, tables, lens)
        out = scaled_cache.paged_attention_scaled(query, k, v, ks, vs, tables, lens)
        eviction.accumulate_attention_weights(query, k, tables, lens, weights, key_scale=ks)
        moved = eviction.evict_by_weight(weights, k, v, tables, lens, new_tables, 48, recent=7,
                                         key_scale=ks, value_scale=vs, into=into)
        return (out * 2, *moved)

    names = ("query", "key", "value", "k", "v", "ks", "vs", "tables", "lens", "weights",
             "new_tables", "into_k", "into_v", "into_ks", "into_vs")
    want, got = _state(40, kv=INT8), _state(40, kv=INT8)
    a = step(*[want[n] for n in names])
    b = torch.compile(step, backend="eager", fullgraph=True)(*[got[n] for n in names])
    assert _equal(a, b)
    assert _equal([want[n] for n in names], [got[n] for n in names])


def test_traced_eviction_in_place():
    """Within one pool and over the weights themselves, also where the trace is made free of
    writes and put back together (aot_eager)."""
    def thin(weights, k, v, ks, vs, tables, lens, new_tables):
        moved = eviction.evict_by_weight(weights, k, v, tables, lens, new_tables, 48, sink=2,
                                         recent=7, key_scale=ks, value_scale=vs,
                                         new_weights=weights)
        return [x * 2 for x in moved]

    names = ("weights", "k", "v", "ks", "vs", "tables", "lens", "new_tables")
    states = [_state(41, kv=INT8) for _ in range(3)]
    for s in states:
        s["new_tables"] = (100 + torch.arange(9)).view(3, 3).to(torch.int32).cuda()
    calls = [thin, *(torch.compile(thin, backend=how, fullgraph=True)
                     for how in ("eager", "aot_eager"))]
    results = [f(*[s[n] for n in names]) for f, s in zip(calls, states)]
    for r, s in zip(results[1:], states[1:]):
        assert _equal(results[0], r)
        assert _equal([states[0][n] for n in names], [s[n] for n in names])


def test_keys_and_values_written_to_one_place_are_refused():
    s = _state(9)
    before = _bits([s["k"], s["v"], s["ks"], s["vs"]])
    for k, v, ks, vs in (("k", "k", "ks", "vs"), ("k", "v", "vs", "vs")):
        with pytest.raises(ValueError, match="of their own"):
            scaled_cache.append_scaled_kv(s["key"], s["value"], s[k], s[v], s[ks], s[vs],
                                          s["tables"], s["lens"])
    for into in (("into_k", "into_k", "into_ks", "into_vs"), ("into_k", "into_v") + 2 * ("into_ks",)):
        with pytest.raises(ValueError, match="of their own"):
            eviction.evict_by_weight(s["weights"], s["k"], s["v"], s["tables"], s["lens"],
                                     s["new_tables"], s["budget"], key_scale=s["ks"],
                                     value_scale=s["vs"], into=tuple(s[n] for n in into))
    assert _equal(before, [s["k"], s["v"], s["ks"], s["vs"]])


def test_a_pool_past_32_bit_offsets():
    """Pages past 4 GiB of a pool, read, written and moved to."""
    page, hkv, d = 64, 8, 128
    pages = (5 << 30) // (page * hkv * d)
    k, v = (torch.zeros(pages, page, hkv, d, dtype=torch.uint8, device="cuda").view(E4M3)
            for _ in range(2))
    ks, vs = (torch.ones(pages, hkv, device="cuda") for _ in range(2))
    lens = torch.tensor([200, 130], dtype=torch.int32)
    tables = torch.tensor([[pages - 1, 3, pages - 2, pages - 9],
                           [pages - 4, pages - 3, 5, 0]], dtype=torch.int32)
    g = torch.Generator().manual_seed(50)
    key, value = (torch.randn(2, 200, hkv, d, generator=g).half() for _ in range(2))
    q = torch.randn(2, 4, 32, d, generator=g).half()
    bt, sl = _cuda(tables, lens)
    scaled_cache.append_scaled_kv(*_cuda(key, value), k, v, ks, vs, bt, sl, new_lens=sl)
    ids = tables.flatten().unique().long()
    small = torch.searchsorted(ids, tables.long()).to(torch.int32)
    pick = ids.cuda()
    caches = [c.view(torch.uint8)[pick].cpu().view(E4M3) for c in (k, v)]
    scales = [s[pick].cpu() for s in (ks, vs)]
    mine = [torch.zeros(len(ids), page, hkv, d, dtype=torch.uint8).view(E4M3) for _ in range(2)]
    mine_s = [torch.ones(len(ids), hkv) for _ in range(2)]
    ref.append(key, value, mine, mine_s, small, lens, lens)
    for a, b in zip(scales, mine_s):
        assert torch.equal(a, b)
    off = sum((a.view(torch.uint8) != b.view(torch.uint8)).sum().item() for a, b in zip(caches, mine))
    assert off < 200 * 8  # ties of the rounding only
    want, bound, mass = ref.attention(q, *caches, *scales, small, lens)
    out = scaled_cache.paged_attention_scaled(q.cuda(), k, v, ks, vs, bt, sl)
    ref.assert_within(out, want, bound)
    weights = torch.zeros(2, hkv, 256, device="cuda")
    eviction.accumulate_attention_weights(q.cuda(), k, bt, sl, weights, key_scale=ks)
    ref.assert_within(weights, *ref.weights_after(torch.zeros(2, hkv, 256), mass, lens, 4))
    new = torch.tensor([[pages - 20, 21], [pages - 22, 23]], dtype=torch.int32)
    got = eviction.evict_by_weight(weights, k, v, bt, sl, new.cuda(), 70, key_scale=ks,
                                   value_scale=vs)
    into = [torch.zeros(4, page, hkv, d, dtype=torch.uint8).view(E4M3) for _ in range(2)]
    into_s = [torch.zeros(4, hkv) for _ in range(2)]
    kept = ref.evict(weights.cpu(), caches, scales, small, lens,
                     torch.arange(4).view(2, 2).to(torch.int32), 70, 0, 0, into, into_s)[2]
    assert torch.equal(got[2].cpu(), kept)
    for c, w, s, ws in zip((k, v), into, (ks, vs), into_s):
        at = new.flatten().long().cuda()
        assert torch.equal(c.view(torch.uint8)[at].cpu(), w.view(torch.uint8))
        assert torch.equal(s[at].cpu(), ws)


def test_scales_of_heads_past_32_bit_offsets():
    """Scales whose heads lie 1 GiB apart: the upper heads' are past 4 GiB of the tensor, and
    each operator reads (and writes) its own head's."""
    hkv, d, page, far = 8, 64, 16, 1 << 28
    lens = [90, 33]
    q, caches, scales, tables, sl = _inputs(lens, 2, 16, hkv, d, page, F16, INT8, 60)
    pages = scales[0].shape[0]
    store = [torch.empty(hkv * far, device="cuda") for _ in range(2)]
    ks, vs = (x.as_strided((pages, hkv), (1, far)) for x in store)
    for x, s in zip((ks, vs), scales):
        x.copy_(s)
    qc, kc, vc, bt, slc = _cuda(q, *caches, tables, sl)
    want, bound, mass = ref.attention(q, *caches, *scales, tables, sl)
    ref.assert_within(scaled_cache.paged_attention_scaled(qc, kc, vc, ks, vs, bt, slc), want, bound)
    weights = torch.zeros(2, hkv, 96, device="cuda")
    eviction.accumulate_attention_weights(qc, kc, bt, slc, weights, key_scale=ks)
    ref.assert_within(weights, *ref.weights_after(torch.zeros(2, hkv, 96), mass, sl, 2))
    new_tables = torch.arange(4).view(2, 2).to(torch.int32)
    into = [torch.zeros(4, page, hkv, d, dtype=INT8) for _ in range(2)]
    into_s = [torch.zeros(4, hkv) for _ in range(2)]
    gi = _cuda(*into)
    gs = [x.as_strided((4, hkv), (1, far), pages) for x in store]
    eviction.evict_by_weight(weights, kc, vc, bt, slc, new_tables.cuda(), 32, key_scale=ks,
                             value_scale=vs, into=(*gi, *gs))
    ref.evict(weights.cpu(), caches, scales, tables, sl, new_tables, 32, 0, 0, into, into_s)
    assert _equal([x.cpu() for x in gi], into)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(gs, into_s))
    g = torch.Generator().manual_seed(61)
    key, value = (torch.randn(2, 3, hkv, d, generator=g).half() for _ in range(2))
    scaled_cache.append_scaled_kv(*_cuda(key, value), kc, vc, ks, vs, bt, slc)
    ref.append(key, value, caches, scales, tables, sl)
    for a, b in zip((ks, vs), scales):
        assert torch.equal(a.cpu().nan_to_num(), b.nan_to_num())


def test_a_wrapper_whose_workspace_fits_one_plan_only():
    """A buffer large enough for the ordinary plan of a short sequence (none at all) serves
    runs over block scales too, captured ones among them; an int8 plan asks for its own."""
    q, caches, scales, tables, sl = _inputs([60], 2, 8, 2, 128, 16, F16, E4M3, 33)
    pool = tuple(_cuda(*caches))
    qc, ks, vs = _cuda(q.view(2, 8, 128), *scales)
    csr = _cuda(torch.tensor([0, 4], dtype=torch.int32), tables[0, :4].contiguous(),
                torch.tensor([12], dtype=torch.int32))
    ws = torch.zeros(16, dtype=torch.uint8, device="cuda")
    want, bound, _ = ref.attention(q, *caches, *scales, tables, sl)
    w = decode_api.BatchDecodeWithPagedKVCacheWrapper(ws, "NHD")
    w.plan(*csr, 8, 2, 128, 16, q_data_type=F16, kv_data_type=E4M3, q_len_per_req=2)
    ref.assert_within(w.run(qc, pool, kv_block_scales=(ks, vs)).view(q.shape), want, bound)
    w.run(qc, pool)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = w.run(qc, pool, kv_block_scales=(ks, vs))
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        ref.assert_within(out.view(q.shape), want, bound)
        w.run(qc, pool, kv_block_scales=(ks, vs))
    assert (ws == 0).all()
    with pytest.raises(ValueError, match="float_workspace_buffer"):
        w.plan(*csr, 8, 2, 128, 16, q_data_type=F16, kv_data_type=INT8, q_len_per_req=2)


def test_host_threads_on_one_stream():
    """Two threads' calls on the default stream, their kernels launched between each other's:
    the bits of the calls made alone."""
    import threading

    lens = ((2500, 77, 513), (300, 1900, 40))
    states = [_state(70 + i, (300, 77, 513)) for i in range(2)]
    for s, n in zip(states, lens):  # long enough for several splits of a sequence
        s["tables"] = s["tables"].repeat(1, 5)[:, :160].contiguous()
        s["lens"].copy_(torch.tensor(n, dtype=torch.int32))

    def call(s):
        w = torch.zeros(3, 2, 2600, device="cuda")
        out = scaled_cache.paged_attention_scaled(*[s[k] for k in (
            "query", "k", "v", "ks", "vs", "tables", "lens")])
        eviction.accumulate_attention_weights(s["query"], s["k"], s["tables"], s["lens"], w,
                                              key_scale=s["ks"])
        return out, w

    want = [call(s) for s in states]
    torch.cuda.synchronize()
    got, errors, start = [[], []], [], threading.Barrier(2)

    def worker(i):
        try:
            start.wait()
            for _ in range(20):
                got[i].append(call(states[i]))
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
        assert len(got[i]) == 20 and all(_equal(g, want[i]) for g in got[i])


def test_lengths_past_the_table_up_to_the_largest():
    """Lengths are held to the table: the largest number there is acts as any other past it."""
    tops = [2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 16]
    b, width = len(tops), 30

    def run(lens):
        s = _state(80, (400,) * b)
        s["tables"] = s["tables"][:, :width].contiguous()
        s["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        return _step(s)

    past = run([width * 16 + 100] * b)
    for a, w in zip(_bits(run(tops)), _bits(past)):
        assert torch.equal(a, w)
    assert (past[0].abs().sum(-1) > 0).all() and (past[1] == 48).all()
