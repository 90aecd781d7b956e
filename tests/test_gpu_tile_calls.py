"""How attention over shared prefixes is called where a group has more rows than a wave holds
(the tile kernels): captured in graphs, on several streams and threads, traced."""

import threading

import pytest

torch = pytest.importorskip("torch")

from small_q_attention_amd.shared_prefix import (paged_attention_shared_prefix,  # noqa: E402
                                                 plan_shared_prefix)
from tests import _part_reference as ref  # noqa: E402
from tests._part_reference import BF16, E4M3, F16, INT8  # noqa: E402
from tests.test_gpu_shared_prefix import p_step  # noqa: E402

pytestmark = pytest.mark.gpu

# 384 and 240 rows of a kv head, in blocks of 256; two sequences of no group.
GROUPS, PAGE, Q, HQ, HKV, BATCH, WIDTH = [(0, 24, 23), (25, 15, 9)], 16, 4, 8, 2, 41, 40
KINDS = [(F16, None, False, 128), (BF16, None, False, 64), (BF16, E4M3, False, 128),
         (F16, INT8, True, 128), (BF16, None, False, 256)]
LENS = [370 + 4 + 6 * i % 200 for i in range(24)] + [300] + \
       [146 + 4 + 11 * i % 300 for i in range(15)] + [17]


def _cpu(seed, kind, lens=LENS):
    dtype, kv, scaled, d = kind
    g = torch.Generator().manual_seed(seed)
    pool = BATCH * WIDTH
    tables = torch.randperm(pool, generator=g).to(torch.int32).view(BATCH, WIDTH)
    for first, count, pages in GROUPS:
        tables[first:first + count, :pages] = tables[first, :pages]
    q = torch.randn(BATCH, Q, HQ, d, generator=g).to(dtype)
    (k, ks), (v, vs) = (ref.cache(pool, PAGE, HKV, d, dtype, kv, scaled, g) for _ in range(2))
    return q, k, v, tables, torch.tensor(lens, dtype=torch.int32), ks, vs


def _state(*a, **kw):
    return ref.cuda(*_cpu(*a, **kw))


def _plan(kind):
    return plan_shared_prefix(GROUPS, BATCH, Q, HQ, HKV, kind[3], PAGE)


def _call(s, plan, **kw):
    return paged_attention_shared_prefix(*s[:5], plan, key_scale=s[5], value_scale=s[6], **kw)


def _load(s, t):
    for a, b in zip(s, t):
        if a is not None:
            a.copy_(b)


@pytest.mark.parametrize("kind", KINDS)
def test_captured_in_a_graph(kind):
    """Replays with other data, lengths among it, give the eager calls' bits, and those are the
    definition's."""
    s, plan = _state(1, kind), _plan(kind)
    _call(s, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _call(s, plan)
    short = [0, 5, 369, 372, 371] + LENS[5:]  # padded sequences; the third to fifth of the group
    for seed, lens in ((2, LENS), (3, [640] * BATCH), (4, short), (5, [0] * BATCH), (6, LENS)):
        host = _cpu(seed, kind, lens)
        want = _call(ref.cuda(*host), plan)
        _load(s, host)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), (seed, lens)
        if lens is short:
            q, k, v, tables, sl, ks, vs = host
            exact, bound = ref.attention(q, k, v, ks, vs, tables, sl,
                                         lambda i, n: ref.window_seen(n, Q, 1 << 30, 0),
                                         p_step=p_step(kind[0], kind[2]))
            ref.assert_within(got, exact, bound)


def test_two_graphs_replayed_at_once():
    kind = KINDS[0]
    plan, states, graphs, outs = _plan(kind), [_state(7, kind), _state(8, kind)], [], []
    for s in states:
        _call(s, plan)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_call(s, plan))
        graphs.append(g)
    want = [_call(s, plan) for s in states]
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("kind", KINDS[:4])
def test_on_several_streams(kind):
    plan = _plan(kind)
    states = [_state(10 + i, kind) for i in range(4)]
    want = [_call(s, plan) for s in states]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in states], []
    for s, st in zip(states, streams):
        with torch.cuda.stream(st):
            outs.append(_call(s, plan))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_host_threads_on_one_stream():
    kind = KINDS[1]
    plan, states = _plan(kind), [_state(20 + i, KINDS[1]) for i in range(2)]
    want = [_call(s, plan) for s in states]
    torch.cuda.synchronize()
    got, errors, start = [[], []], [], threading.Barrier(2)

    def worker(i):
        try:
            start.wait()
            for _ in range(20):
                got[i].append(_call(states[i], plan))
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
        assert len(got[i]) == 20 and all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("kind", KINDS[:4])
def test_traced(kind):
    plan, s = _plan(kind), _state(30, kind)

    def step(q, k, v, tables, lens, ks, vs):
        return paged_attention_shared_prefix(q, k, v, tables, lens, plan, key_scale=ks,
                                             value_scale=vs) * 2

    assert torch.equal(torch.compile(step, backend="aot_eager", fullgraph=True)(*s), step(*s))
