"""Attention over part of a cache, and over a cache that sequences share: how the two
operators are called, and what they compute.

* ``window``: small-q attention whose rows see the last tokens before them and the first
  few of their sequence;
* ``prefix``: small-q attention of a batch whose sequences begin with the same pages, group
  by group, computed once for each group.

Fields of a case: ``op``; ``batch``; ``q_len`` (draft rows); ``lo``, ``hi``: lengths spread
evenly over the batch and dealt in an order of the seed (for ``prefix`` what follows the
shared pages, draft tokens included); ``hq``, ``hkv``, ``d``, ``page``; ``dtype`` of the
queries; ``kv``: the cache's element type (``int8`` and ``scaled``: codes with one scale for
each page and kv head); ``tree``: a draft tree per request instead of the draft chain;
``window``, ``sink``; ``groups``: groups of a ``prefix`` batch, the first of them the
smallest, whose shared tokens lie between ``shared_lo`` and ``shared_hi``.
"""

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn,
          "int8": torch.int8}
CODE_MAX = {"e4m3": 448.0, "int8": 127.0}
POOL = 1.125  # pages of a pool over pages in use: a serving engine keeps some free


def _case(name, op, batch, q_len, lo, hi, *, hq=32, hkv=8, d=128, page=16, dtype="fp16", kv="",
          scaled=False, tree=False, window=0, sink=0, groups=0, shared_lo=0, shared_hi=0):
    return {"name": name, "op": op, "batch": batch, "q_len": q_len, "lo": lo, "hi": hi,
            "hq": hq, "hkv": hkv, "d": d, "page": page, "dtype": dtype, "kv": kv or dtype,
            "scaled": scaled, "tree": tree, "window": window, "sink": sink, "groups": groups,
            "shared_lo": shared_lo, "shared_hi": shared_hi}


def listed():
    return [
        # One short conversation through a layer of a small window, the next token: latency.
        _case("window_one_1k_q1", "window", 1, 1, 1021, 1021, window=128, sink=4),
        # One long stream that keeps its first tokens and the last 4K, four draft tokens.
        _case("window_one_128k_q4", "window", 1, 4, 131072, 131072, window=4096, sink=16),
        # A serving batch as it comes, some sequences shorter than the window, draft trees,
        # integer codes with block scales under bf16 queries.
        _case("window_ragged_24_q4_int8", "window", 24, 4, 517, 16111, page=64, dtype="bf16",
              kv="int8", scaled=True, tree=True, window=2048, sink=64),
        # Narrow heads, eight queries to a kv head, no first tokens.
        _case("window_40x8k_d64_bf16", "window", 40, 2, 6007, 8191, hq=64, d=64, dtype="bf16",
              window=1024),
        # Long contexts at a decoding batch, e4m3 under one scale per tensor.
        _case("window_100x32k_q1_e4m3", "window", 100, 1, 32749, 32768, kv="e4m3", window=4096,
              sink=4),
        # The same length as the benchmark's cfg3, eight draft tokens.
        _case("window_64x32k_q8", "window", 64, 8, 32768, 32768, window=4096, sink=4),
        # Eight answers to one prompt, sampled side by side: latency.
        _case("prefix_8x2k_q1", "prefix", 8, 1, 33, 190, groups=1, shared_lo=2048,
              shared_hi=2048),
        # A serving batch under five system prompts, three draft tokens each, e4m3.
        _case("prefix_41_in_5_q3_e4m3", "prefix", 41, 3, 61, 2003, page=64, dtype="bf16",
              kv="e4m3", groups=5, shared_lo=1088, shared_hi=8128),
        # Wide heads, bf16, draft trees below one prompt.
        _case("prefix_24x4k_d256_bf16", "prefix", 24, 5, 77, 700, hq=16, hkv=4, d=256,
              page=32, dtype="bf16", tree=True, groups=1, shared_lo=4096, shared_hi=4096),
        # A decoding batch under one long document, a token at a time.
        _case("prefix_64x16k_q1", "prefix", 64, 1, 129, 1031, groups=1, shared_lo=16384,
              shared_hi=16384),
        # The same in bf16 with four draft tokens, two documents.
        _case("prefix_96_in_2_q4_bf16", "prefix", 96, 4, 250, 2047, dtype="bf16", groups=2,
              shared_lo=8192, shared_hi=16384),
        # Many requests over one context of 32K, eight draft tokens each.
        _case("prefix_64x32k_q8", "prefix", 64, 8, 500, 1024, groups=1, shared_lo=32768,
              shared_hi=32768),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["window", "prefix"])
    hkv = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 4, 4, 8])
    d = rng.choice([64, 128, 128, 256])
    most = min(16, (32 if d == 256 else 64) // group)
    dtype = rng.choice(["fp16", "bf16"])
    page = rng.choice([16, 16, 32, 64, 256])
    q_len = rng.randint(1, most)
    kw = dict(hq=hkv * group, hkv=hkv, d=d, page=page, dtype=dtype, tree=rng.random() < 0.3)
    token = hkv * d
    if op == "window":
        kv, scaled = rng.choice([(dtype, False), (dtype, False), ("e4m3", False), ("e4m3", True),
                                 ("int8", True)])
        batch, hi, window = log(1, 128), log(64, 131072), log(16, 8192)
        sink = rng.choice([0, 0, 1, 4, 16, 100])
        lo = hi if rng.random() < 0.5 else max(q_len, hi // rng.choice([2, 8]))
        while batch > 1 and batch * min(hi, window + sink + q_len) * token > 64 * 4108 * 1024:
            batch = max(1, batch * 3 // 4)
        case = _case("", op, batch, q_len, hi if batch == 1 else max(lo, q_len), max(hi, q_len),
                     kv=kv, scaled=scaled, window=window, sink=sink, **kw)
    else:
        batch = log(2, 128)
        groups = rng.choice([1, 1, 2, max(1, batch // 8)])
        shared_hi = max(page, log(128, 32768) // page * page)
        shared_lo = shared_hi if rng.random() < 0.5 else max(page, shared_hi // 4 // page * page)
        own_hi = log(max(q_len, 8), 2048)
        own_lo = max(q_len, own_hi // rng.choice([1, 2, 16]))
        # Within the cost of the largest listed case: its products, and its own tokens.
        while batch > 2 and (batch * q_len * group * shared_hi * token
                             > 64 * 8 * 4 * 32768 * 1024 * 9 // 10
                             or batch * own_hi * token > 64 * 1024 * 1024):
            batch = max(2, batch * 3 // 4)
        case = _case("", op, batch, q_len, own_lo, own_hi, kv=rng.choice([dtype, dtype, "e4m3"]),
                     groups=min(groups, batch), shared_lo=shared_lo, shared_hi=shared_hi, **kw)
    del case["name"]
    return case


def _spread(lo, hi, n):
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _groups(case):
    """(first, count, shared tokens) of every group: sizes 1 : 2 : 3 : ..., rounded down,
    the rest in the last one; with 8 sequences, of 3 groups, 1, 2 and 5."""
    n, b, page = case["groups"], case["batch"], case["page"]
    sizes = [max(1, 2 * b * (i + 1) // (n * (n + 1))) for i in range(n)]
    while sum(sizes[:-1]) >= b:  # many small groups
        sizes = [max(1, x - 1) for x in sizes]
        if max(sizes) == 1:
            break
    sizes[-1] = b - sum(sizes[:-1])
    shared = [x // page * page for x in _spread(case["shared_lo"], case["shared_hi"], n)]
    first = [sum(sizes[:i]) for i in range(n)]
    return list(zip(first, sizes, shared))


def _live(n, case):
    """Pages of a sequence of n tokens that some row sees: (first tokens', the last ones')."""
    page = case["page"]
    pages = -(-n // page)
    head = min(-(-case["sink"] // page), pages)
    tail = max(n - case["q_len"] + 1 - case["window"], 0) // page
    return head, max(tail, head), pages


def _deal(values, gen):
    return torch.tensor(values)[torch.randperm(len(values), generator=gen)]


def _tokens(g, *shape, dtype):
    """Keys and values as they come: a few tokens stand out, as attention sinks and
    rare words do (four times the others, one in a hundred)."""
    x = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    hit = torch.rand(*shape[:-2], 1, 1, generator=g, device="cuda") < 0.01
    return x.mul_(torch.where(hit, 4.0, 1.0).to(dtype))


def _pool(g, pages, case):
    """One pool [pages, page, Hkv, D] in the cache's type, and its scales [pages, Hkv]
    (None without block scales)."""
    half = DTYPES[case["dtype"]]
    x = _tokens(g, pages, case["page"], case["hkv"], case["d"], dtype=half)
    if not case["scaled"]:
        return x.to(DTYPES[case["kv"]]), None
    most = CODE_MAX[case["kv"]]
    scale = x.abs().amax((1, 3)).float() / most
    for part in torch.arange(pages, device="cuda").split(4096):  # bounded temporaries
        y = x[part].float() / scale[part][:, None, :, None]
        x[part] = (y.round() if case["kv"] == "int8" else y).clamp(-most, most).to(half)
    return x.to(DTYPES[case["kv"]]), scale


def _trees(b, q_len, gen):
    """Each draft token hangs below an earlier one; a row sees its ancestors."""
    parent = torch.rand(b, q_len, generator=gen)
    seen = torch.zeros(b, q_len, q_len, dtype=torch.bool)
    for i in range(q_len):
        seen[:, i, i] = True
        if i:
            seen[:, i] |= seen[torch.arange(b), (parent[:, i] * i).long()]
    return seen.cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    gh = torch.Generator().manual_seed(int(seed))
    b, q_len, hq, hkv, d, page = (case[k] for k in ("batch", "q_len", "hq", "hkv", "d", "page"))
    lens = _deal(_spread(case["lo"], case["hi"], b), gh)
    groups = []
    if case["op"] == "prefix":
        groups = _groups(case)
        for first, count, shared in groups:
            lens[first:first + count] += shared
    width = -(-int(lens.max()) // page)
    tables = torch.full((b, width), -1, dtype=torch.int32)
    # Pages of a pool in shuffled order: those a window has left behind are gone, those of a
    # shared prefix are there once.
    rows = []
    if case["op"] == "window":
        for i, n in enumerate(lens.tolist()):
            head, tail, pages = _live(n, case)
            rows.append((i, i + 1, torch.cat([torch.arange(head), torch.arange(tail, pages)])))
    else:
        for first, count, shared in groups:
            rows.append((first, first + count, torch.arange(shared // page)))
            for i in range(first, first + count):
                rows.append((i, i + 1, torch.arange(shared // page, -(-int(lens[i]) // page))))
    used = sum(len(at) for _, _, at in rows)
    pool = int(math.ceil(used * POOL))
    perm = torch.randperm(pool, generator=gh).to(torch.int32)
    taken = 0
    for first, last, at in rows:
        tables[first:last, at] = perm[taken:taken + len(at)]
        taken += len(at)
    half = DTYPES[case["dtype"]]
    s = {"op": case["op"], "page": page, "tables": tables.cuda(), "scale": d ** -0.5,
         "lens": lens.to(torch.int32).cuda(), "most": int(lens.max()), "groups": groups,
         "window": case["window"], "sink": case["sink"], "own_most": case["hi"]}
    s["k"], s["k_scale"] = _pool(g, pool, case)
    s["v"], s["v_scale"] = _pool(g, pool, case)
    s["query"] = torch.randn(b, q_len, hq, d, generator=g, device="cuda", dtype=half)
    s["trees"] = _trees(b, q_len, gh) if case["tree"] else None
    if own:
        from small_q_attention_amd import masks

        s["mask"] = masks.pack_draft_mask(s["trees"]) if s["trees"] is not None else None
        if groups:
            from small_q_attention_amd import shared_prefix

            s["plan"] = shared_prefix.plan_shared_prefix(
                [(first, count, shared // page) for first, count, shared in groups], batch=b,
                q_len=q_len, num_query_heads=hq, num_kv_heads=hkv, head_dim=d, page_size=page)
    return s


def run(s):
    return OPERATORS[s["op"]][1 if own else 0](s)


# The framework's calls.

def _window_own(s):
    from small_q_attention_amd import windowed

    return windowed.paged_attention_windowed(
        s["query"], s["k"], s["v"], s["tables"], s["lens"], s["window"], sink=s["sink"],
        key_scale=s["k_scale"], value_scale=s["v_scale"], max_seq_len=s["most"], mask=s["mask"])


def _prefix_own(s):
    from small_q_attention_amd import shared_prefix

    return shared_prefix.paged_attention_shared_prefix(
        s["query"], s["k"], s["v"], s["tables"], s["lens"], s["plan"], max_seq_len=s["most"],
        mask=s["mask"])


# The plain forms.

def _bytes(x):
    return x.view(torch.uint8) if x.element_size() == 1 else x


def _gather(cache, scale, tables, at, page):
    """Tokens at positions ``at`` [B, n] (negative: none), [B, Hkv, n, D] in 32 bits."""
    at = at.clamp(min=0)
    ids = tables.long().gather(1, at // page).clamp(min=0)
    x = _bytes(cache)[ids, at % page].view(cache.dtype).float()
    if scale is not None:
        x = x * scale[ids][..., None]
    return x.transpose(1, 2).contiguous()


def _by_kv_head(s):
    """The queries as [B, Hkv, Q * G, D] in 32 bits."""
    q = s["query"].float()
    b, q_len, hq, d = q.shape
    hkv = s["k"].shape[2]
    return q.view(b, q_len, hkv, hq // hkv, d).transpose(1, 2).reshape(b, hkv, -1, d)


def _back(o, query):
    b, q_len, hq, d = query.shape
    hkv = o.shape[1]
    o = o.view(b, hkv, q_len, hq // hkv, d).transpose(1, 2).reshape(b, q_len, hq, d)
    return o.to(query.dtype)


def _sees(s, at):
    """[B, Q, n]: which tokens at positions ``at`` [B, n] draft row i sees of its draft block
    and of what lies before it."""
    b, q_len = s["query"].shape[:2]
    draft = at - (s["lens"].long()[:, None] - q_len)  # index in the draft block
    if s["trees"] is None:
        chain = torch.ones(q_len, q_len, dtype=torch.bool, device=at.device).tril()
        trees = chain[None].expand(b, -1, -1)
    else:
        trees = s["trees"]
    index = draft.clamp(0, q_len - 1)[:, None].expand(-1, q_len, -1)
    inside = (at >= 0) & (draft < q_len)
    return ((draft < 0)[:, None] | trees.gather(2, index)) & inside[:, None]


def _softmax_parts(scores, seen):
    """Row maxima, exponentials and their sums over what a row sees."""
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    e = torch.exp(scores - top)
    return top, e, e.sum(-1, keepdim=True)


def _window_plain(s):
    q, lens, group = _by_kv_head(s), s["lens"].long(), s["query"].shape[2] // s["k"].shape[2]
    q_len, window, sink = s["query"].shape[1], s["window"], s["sink"]
    reach = min(window + q_len - 1, s["most"])  # tokens up to the end that some row sees
    first = torch.arange(min(sink, s["most"]), device=q.device)[None].expand(len(lens), -1)
    last = lens[:, None] - reach + torch.arange(reach, device=q.device)[None]
    first = torch.where(first < torch.minimum(lens[:, None], last[:, :1]), first, -1)
    at = torch.cat([first, last], 1)
    row = lens[:, None] - q_len + torch.arange(q_len, device=q.device)[None]
    seen = _sees(s, at) & ((at[:, None] < sink) | (at[:, None] > (row - window)[:, :, None]))
    seen = seen.repeat_interleave(group, 1)[:, None]
    k = _gather(s["k"], s["k_scale"], s["tables"], at, s["page"])
    scores = q @ k.transpose(2, 3).contiguous() * s["scale"]
    _, e, total = _softmax_parts(scores, seen)
    del scores, k
    v = _gather(s["v"], s["v_scale"], s["tables"], at, s["page"])
    return _back(torch.where(total > 0, (e @ v) / total, 0.0), s["query"])


def _prefix_plain(s):
    q, lens, group = _by_kv_head(s), s["lens"].long(), s["query"].shape[2] // s["k"].shape[2]
    b, hkv, rows, d = q.shape
    page, n = s["page"], s["own_most"]
    start = torch.zeros(b, dtype=torch.long, device=q.device)
    for first, count, shared in s["groups"]:
        start[first:first + count] = shared
    # What follows the shared pages, sequence by sequence ...
    at = start[:, None] + torch.arange(n, device=q.device)[None]
    at = torch.where(at < lens[:, None], at, -1)
    seen = _sees(s, at).repeat_interleave(group, 1)[:, None]
    k = _gather(s["k"], s["k_scale"], s["tables"], at, page)
    scores = q @ k.transpose(2, 3).contiguous() * s["scale"]
    top, e, total = _softmax_parts(scores, seen)
    o = e @ _gather(s["v"], s["v_scale"], s["tables"], at, page)
    # ... and the shared ones, group by group, joined with it.
    out = torch.empty_like(o)
    for first, count, shared in s["groups"]:
        part = slice(first, first + count)
        at = torch.arange(shared, device=q.device)[None]
        tables = s["tables"][first:first + 1]
        qg = q[part].transpose(0, 1).reshape(hkv, count * rows, d)
        k = _gather(s["k"], s["k_scale"], tables, at, page)[0]
        scores = qg @ k.transpose(1, 2).contiguous() * s["scale"]
        top_g = scores.amax(-1, keepdim=True)
        e_g = torch.exp(scores - top_g)
        del scores
        v = _gather(s["v"], s["v_scale"], tables, at, page)[0]
        total_g, o_g = (x.view(hkv, count, rows, -1).transpose(0, 1)
                        for x in (e_g.sum(-1, keepdim=True), e_g @ v))
        top_g = top_g.view(hkv, count, rows, 1).transpose(0, 1)
        high = torch.maximum(top[part], top_g)
        w, w_g = torch.exp(top[part] - high), torch.exp(top_g - high)
        out[part] = (o[part] * w + o_g * w_g) / (total[part] * w + total_g * w_g)
    return _back(out, s["query"])


OPERATORS = {"window": (_window_plain, _window_own), "prefix": (_prefix_plain, _prefix_own)}


def work(case):
    """Each input read once, each output written once; of a cache the tokens that some row
    sees, a shared prefix once for its group."""
    lens = _spread(case["lo"], case["hi"], case["batch"])
    es = 1 if case["kv"] in CODE_MAX else 2
    b, q, hq, hkv, d, page = (case[k] for k in ("batch", "q_len", "hq", "hkv", "d", "page"))
    if case["op"] == "window":
        w, sink = case["window"], case["sink"]
        read = sum(min(n, w + q - 1 + min(sink, max(n - w - q + 1, 0))) for n in lens)
        seen = 0
        for n in lens:
            for p in range(n - q, n):
                seen += min(p + 1, w + min(sink, max(p + 1 - w, 0)))
    else:
        groups = _groups(case)
        read = sum(lens) + sum(shared for _, _, shared in groups)
        seen = sum(q * n - q * (q - 1) // 2 for n in lens)  # the draft chain
        seen += q * sum(count * shared for _, count, shared in groups)
    scales = 4.0 / (page * d) if case["scaled"] else 0.0  # of an element
    return {"bytes": 2 * read * hkv * d * (es + scales) + 4 * b * q * hq * d
            + 4 * b + 4 * read // page, "flops": 4 * hq * d * seen}


# The definition in 64 bits, sequence by sequence over its own table row.

def exact(case, seed):
    s = prepare(case, seed)
    b, q_len, hq, d = s["query"].shape
    hkv, page = s["k"].shape[2], s["page"]
    out = torch.zeros(b, q_len, hq, d, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lens"].tolist()):
        see = torch.ones(q_len, n, dtype=torch.bool, device="cuda")
        see[:, n - q_len:] = (torch.ones_like(see[:, :q_len]).tril() if s["trees"] is None
                              else s["trees"][i])
        if case["op"] == "window":
            t = torch.arange(n, device="cuda")
            for r in range(q_len):
                see[r] &= (t < case["sink"]) | (t >= n - q_len + r + 1 - case["window"])
        pos = see.any(0).nonzero()[:, 0]
        see = see[:, pos]
        ids = s["tables"][i].long()[pos // page]
        k, v = (_bytes(s[x])[ids, pos % page].view(s[x].dtype).double() for x in ("k", "v"))
        if case["scaled"]:
            k, v = k * s["k_scale"][ids].double()[..., None], v * s["v_scale"][ids].double()[..., None]
        for h in range(hkv):
            q = s["query"][i, :, h * (hq // hkv):(h + 1) * (hq // hkv)].double()
            z = (q.reshape(-1, d) @ k[:, h].t().contiguous()).view(q_len, -1, len(pos)) / math.sqrt(d)
            z = z.masked_fill(~see[:, None], float("-inf"))
            p = torch.softmax(z, -1)
            out[i, :, h * (hq // hkv):(h + 1) * (hq // hkv)] = \
                (p.view(-1, len(pos)) @ v[:, h].contiguous()).view(q_len, -1, d)
    return out
