"""The operators around the paged KV cache: how they are called, and what they compute.

Four operators of a serving engine's cache, each at the sizes of this repository's
benchmark, matrix and tests, with odd and ragged ones among them:

* ``append``: the quantising write into a cache held in 8 bits with one scale for
  each page and kv head;
* ``attend``: small-q attention over such a cache;
* ``weigh``: the attention weight every cached token receives, added up over calls;
* ``evict``: the lighter tokens dropped, the others moved together on new pages.

Fields of a case: ``op``; ``batch``; ``q_len`` (draft rows; for ``append`` the most
new tokens of a sequence); ``lo``, ``hi``: lengths spread evenly over the batch and
dealt in an order of the seed; ``new_lo``: the fewest new tokens of an ``append``
(``q_len``: all sequences alike); ``hq``, ``hkv``, ``d``, ``page``; ``dtype`` of the
queries, of ``append``'s tokens and of 16-bit caches; ``kv``: the cache's element type;
``tree``: a draft tree per request instead of the draft chain; ``budget``, ``sink``,
``recent`` of an ``evict``.
"""

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn,
          "int8": torch.int8}
CODE_MAX = {"e4m3": 448.0, "int8": 127.0}
POOL = 1.125  # pages of a pool over pages in use: a serving engine keeps some free


def _case(name, op, batch, q_len, lo, hi, *, new_lo=0, hq=32, hkv=8, d=128, page=16, dtype="fp16",
          kv="e4m3", tree=False, budget=0, sink=0, recent=0):
    return {"name": name, "op": op, "batch": batch, "q_len": q_len, "lo": lo, "hi": hi,
            "new_lo": new_lo or q_len, "hq": hq, "hkv": hkv, "d": d, "page": page,
            "dtype": dtype, "kv": kv, "tree": tree, "budget": budget, "sink": sink,
            "recent": recent}


def listed():
    return [
        # Every sequence of a decoding batch writes its next four tokens.
        _case("append_decode_32_q4", "append", 32, 4, 1031, 8191, dtype="bf16"),
        # Chunks of eight prompts, uneven, each from the middle of a page on.
        _case("append_chunk_ragged_8", "append", 8, 509, 700, 6007, new_lo=37, page=64),
        # Two prompts of 16K tokens written at once.
        _case("append_prompt_2x16k", "append", 2, 16384, 16384, 16384),
        # One short conversation, the next token: all latency.
        _case("attend_one_1k_q1", "attend", 1, 1, 1024, 1024),
        # A serving batch as it comes, four draft tokens, int8 codes under bf16 queries.
        _case("attend_ragged_24_q4_int8", "attend", 24, 4, 517, 16111, page=64, dtype="bf16",
              kv="int8"),
        # Long contexts at a serving batch, eight draft tokens (the benchmark's cfg3).
        _case("attend_16x32k_q8", "attend", 16, 8, 32768, 32768),
        # One conversation of 2K, a token at a time, over a 16-bit cache.
        _case("weigh_one_2k_q1", "weigh", 1, 1, 2048, 2048, kv="fp16"),
        # Prompts weighed by their last sixteen tokens before they are thinned out.
        _case("weigh_window_ragged_8_q16", "weigh", 8, 16, 1021, 12277, dtype="bf16"),
        # A decoding batch of long contexts over a 16-bit cache.
        _case("weigh_16x32k_q1", "weigh", 16, 1, 32768, 32768, kv="fp16"),
        # One conversation of 8K thinned out to 1K.
        _case("evict_one_8k", "evict", 1, 0, 8191, 8191, kv="fp16", budget=1024, sink=4,
              recent=128),
        # A batch of medium contexts, half of each kept, 64-token pages.
        _case("evict_32x4k_bf16", "evict", 32, 0, 3001, 4099, kv="bf16", dtype="bf16", page=64,
              budget=2000, recent=256),
        # Long ragged contexts of an 8-bit cache thinned out to 4K, some shorter than that.
        _case("evict_ragged_16_e4m3", "evict", 16, 0, 2999, 32749, budget=4096, sink=16,
              recent=512),
    ]


def _lengths(case):
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _new(case):
    """New tokens of each sequence of an append (dealt as the lengths are)."""
    b, lo, hi = case["batch"], case["new_lo"], case["q_len"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["append", "attend", "weigh", "evict"])
    hkv = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 4, 4, 8])
    d = rng.choice([64, 128, 128, 256])
    most = min(16, (32 if d == 256 else 64) // group)
    dtype = rng.choice(["fp16", "bf16"])
    page = rng.choice([16, 16, 32, 64, 256])
    batch, hi = log(1, 48), log(64, 32768)
    lo = hi if rng.random() < 0.4 else max(most, hi // rng.choice([2, 4, 16]))
    kw = dict(hq=hkv * group, hkv=hkv, d=d, page=page, dtype=dtype)
    kv = rng.choice(["e4m3", "int8"]) if op == "attend" else "e4m3"
    q_len = rng.randint(1, most) if op in ("attend", "weigh") else 0
    # A batch within the cost of the largest listed case: its tokens, and their scores.
    while batch > 1 and batch * hi * hkv * (d + 4 * q_len * group) > 14 * 32768 * 8 * 256:
        batch = max(1, batch * 3 // 4)
    if batch == 1:
        lo = hi
    if op == "append":
        q_len = min(lo, log(1, 16384))
        while batch > 1 and batch * q_len * hkv * d > 2 * 16384 * 8 * 128 * 9 // 10:
            batch = max(1, batch * 3 // 4)
        if batch == 1:
            lo = hi
        if hkv * d * q_len * batch > 2 * 16384 * 8 * 128 * 9 // 10:
            q_len = max(1, q_len // 2)
        new_lo = q_len if rng.random() < 0.5 else max(1, q_len // rng.choice([2, 8]))
        case = _case("", op, batch, q_len, lo, hi, new_lo=new_lo, **kw)
    elif op == "evict":
        kv = rng.choice([dtype, "e4m3"])
        budget = max(16, hi // rng.choice([2, 3, 8]) + rng.randint(-7, 7))
        sink = rng.choice([0, 0, 4, 13]) if budget >= 64 else 0
        recent = budget // rng.choice([2, 4, 16])
        case = _case("", op, batch, 0, lo, hi, kv=kv, budget=budget, sink=sink, recent=recent,
                     **kw)
    else:
        if op == "weigh":
            kv = rng.choice([dtype, dtype, "e4m3"])
        case = _case("", op, batch, q_len, max(lo, q_len), max(hi, q_len), kv=kv,
                     tree=rng.random() < 0.4, **kw)
    del case["name"]
    return case


def _deal(values, gen):
    return torch.tensor(values)[torch.randperm(len(values), generator=gen)]


def _tables(used, page_base, pool, width, gen):
    """A block table over shuffled pages of a pool, `used` pages a row."""
    perm = torch.randperm(pool, generator=gen).to(torch.int32) + page_base
    tables = torch.zeros(len(used), width, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used.tolist()):
        tables[i, :n] = perm[at:at + n]
        at += n
    return tables


def _tokens(g, *shape, dtype):
    """Keys and values as they come: a few tokens stand out, as attention sinks and
    rare words do (four times the others, one in a hundred)."""
    x = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    hit = torch.rand(*shape[:-2], 1, 1, generator=g, device="cuda") < 0.01
    return x.mul_(torch.where(hit, 4.0, 1.0).to(dtype))


def _pool(g, pages, case):
    """One pool [pages, page, Hkv, D] in the cache's type, and its scales [pages, Hkv]
    (None for 16-bit caches)."""
    half = DTYPES[case["dtype"]]
    x = _tokens(g, pages, case["page"], case["hkv"], case["d"], dtype=half)
    if case["kv"] not in CODE_MAX:
        return x, None
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
    b, q_len, hkv, d, page = (case[k] for k in ("batch", "q_len", "hkv", "d", "page"))
    lens = _deal(_lengths(case), gh)
    used = (lens + page - 1) // page
    pool = int(math.ceil(int(used.sum()) * POOL))
    width = int(used.max())
    tables = _tables(used, 0, pool, width, gh).cuda()
    s = {"op": case["op"], "page": page, "tables": tables, "lens": lens.to(torch.int32).cuda(),
         "most": case["hi"], "scale": d ** -0.5, "code": CODE_MAX.get(case["kv"])}
    s["k"], s["k_scale"] = _pool(g, pool, case)
    half = DTYPES[case["dtype"]]
    if case["op"] != "weigh":
        s["v"], s["v_scale"] = _pool(g, pool, case)
    if case["op"] == "append":
        s["key"] = _tokens(g, b, q_len, hkv, d, dtype=half)
        s["value"] = _tokens(g, b, q_len, hkv, d, dtype=half)
        new = _deal(_new(case), gh)
        s["new"] = torch.minimum(new, lens).to(torch.int32).cuda()
    elif case["op"] == "evict":
        # Weights as attention leaves them: a few heavy tokens, many light ones, and
        # some that no row ever looked at (ties).
        u = torch.rand(b, hkv, width * page, generator=g, device="cuda")
        s["weights"] = torch.where(u < 0.05, 0.0, (1.0 - u).clamp(min=1e-7).log().square())
        s["budget"], s["sink"], s["recent"] = case["budget"], case["sink"], case["recent"]
        kept = torch.minimum(lens, torch.tensor(case["budget"]))
        used = (kept + page - 1) // page
        into = int(used.sum())
        s["new_tables"] = _tables(used, 0, into, int(used.max()), gh).cuda()
        shape = (into, page, hkv, d)
        s["new_k"] = torch.zeros(shape, dtype=torch.uint8 if s["code"] else half, device="cuda")
        s["new_v"] = torch.zeros_like(s["new_k"])
        s["new_k_scale"] = s["new_v_scale"] = None
        if s["code"]:
            s["new_k"], s["new_v"] = (s[n].view(DTYPES[case["kv"]]) for n in ("new_k", "new_v"))
            s["new_k_scale"] = torch.zeros(into, hkv, device="cuda")
            s["new_v_scale"] = torch.zeros(into, hkv, device="cuda")
    else:
        s["query"] = torch.randn(b, q_len, case["hq"], d, generator=g, device="cuda", dtype=half)
        s["trees"] = _trees(b, q_len, gh) if case["tree"] else None
        if case["op"] == "weigh":
            s["weights"] = torch.rand(b, hkv, width * page, generator=g, device="cuda")
    if own:
        from small_q_attention_amd import _lib, masks

        _lib.load()
        s["mask"] = masks.pack_draft_mask(s["trees"]) if s.get("trees") is not None else None
    return s


def run(s):
    return OPERATORS[s["op"]][1 if own else 0](s)


# The framework's calls.

def _append_own(s):
    from small_q_attention_amd import scaled_cache

    scaled_cache.append_scaled_kv(s["key"], s["value"], s["k"], s["v"], s["k_scale"], s["v_scale"],
                                  s["tables"], s["lens"], new_lens=s["new"])
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _attend_own(s):
    from small_q_attention_amd import scaled_cache

    return scaled_cache.paged_attention_scaled(
        s["query"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["tables"], s["lens"],
        max_seq_len=s["most"], mask=s["mask"])


def _weigh_own(s):
    from small_q_attention_amd import eviction

    return eviction.accumulate_attention_weights(
        s["query"], s["k"], s["tables"], s["lens"], s["weights"], key_scale=s["k_scale"],
        max_seq_len=s["most"], mask=s["mask"])


def _evict_own(s):
    from small_q_attention_amd import eviction

    lens, weights, kept = eviction.evict_by_weight(
        s["weights"], s["k"], s["v"], s["tables"], s["lens"], s["new_tables"], s["budget"],
        sink=s["sink"], recent=s["recent"], key_scale=s["k_scale"], value_scale=s["v_scale"],
        into=(s["new_k"], s["new_v"], s["new_k_scale"], s["new_v_scale"]))
    return (lens, weights, kept, s["new_k"], s["new_v"], s["new_k_scale"], s["new_v_scale"])


# The plain forms.

def _bytes(x):
    return x.view(torch.uint8) if x.element_size() == 1 else x


def _gather(cache, scale, tables):
    """Tokens of every sequence, [B, tokens, Hkv, D] in 32 bits."""
    ids = tables.long()
    x = _bytes(cache)[ids].view(cache.dtype).float()
    if scale is not None:
        x = x * scale[ids][:, :, None, :, None]
    return x.flatten(1, 2)


def _probabilities(s):
    """Softmax probabilities [B, Hkv, Q * G, tokens]: token t of a sequence is seen by
    draft row i if it lies before the draft block or is a draft token the row sees."""
    q = s["query"].float()
    b, q_len, hq, d = q.shape
    k = _gather(s["k"], s["k_scale"], s["tables"])
    tokens, hkv = k.shape[1], k.shape[2]
    q = q.view(b, q_len, hkv, hq // hkv, d).transpose(1, 2).reshape(b, hkv, -1, d)
    scores = q @ k.permute(0, 2, 3, 1).contiguous() * s["scale"]
    at = torch.arange(tokens, device=q.device)
    draft = at[None] - (s["lens"].long()[:, None] - q_len)  # index in the draft block
    if s["trees"] is None:
        chain = torch.ones(q_len, q_len, dtype=torch.bool, device=q.device).tril()
        trees = chain[None].expand(b, -1, -1)
    else:
        trees = s["trees"]
    index = draft.clamp(0, q_len - 1)[:, None].expand(-1, q_len, -1)
    seen = (draft < 0)[:, None] | (trees.gather(2, index) & (draft < q_len)[:, None])
    seen = seen.repeat_interleave(hq // hkv, 1)[:, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0), draft


def _attend_plain(s):
    p, draft = _probabilities(s)
    b, q_len, hq, d = s["query"].shape
    v = _gather(s["v"], s["v_scale"], s["tables"])
    v = torch.where((draft < q_len)[:, :, None, None], v, 0.0)
    o = p @ v.transpose(1, 2).contiguous()
    o = o.view(b, v.shape[2], q_len, -1, d).transpose(1, 2).reshape(b, q_len, hq, d)
    return o.to(s["query"].dtype)


def _weigh_plain(s):
    p, draft = _probabilities(s)
    p = p.sum(2)
    q_len, tokens = s["query"].shape[1], p.shape[2]
    old = s["weights"][:, :, :tokens]
    draft = draft[:, None]
    new = torch.where(draft < 0, old + p, torch.where(draft < q_len, p, old))
    s["weights"][:, :, :tokens] = new
    return s["weights"]


def _encode(x, scale, dtype, most):
    y = torch.where(scale > 0, x / scale, 0.0)
    return (y.round() if dtype is torch.int8 else y).clamp(-most, most).to(dtype)


def _append_plain(s):
    b, q_len = s["key"].shape[:2]
    page, pages, most = s["page"], s["k"].shape[0], s["code"]
    lens, new = s["lens"].long(), s["new"].long()
    rows = torch.arange(b, device=lens.device)[:, None]
    # Past a sequence's new tokens its last one again: the same write.
    i = torch.minimum(torch.arange(q_len, device=lens.device)[None], new[:, None] - 1)
    at = (lens - new)[:, None] + i
    ids = s["tables"].long().gather(1, at // page)
    slot = at % page
    touched = torch.zeros(pages, dtype=torch.bool, device=lens.device)
    touched[ids.flatten()] = True
    # A page that holds earlier tokens of its sequence keeps a scale for them too.
    first, before = ids[:, 0], (lens - new) % page
    held = torch.zeros(pages, dtype=torch.bool, device=lens.device)
    held[first] = before > 0
    for x, cache, scale in ((s["key"], s["k"], s["k_scale"]), (s["value"], s["v"], s["v_scale"])):
        x = x[rows, i].float()
        top = x.abs().amax(-1).flatten(0, 1)
        want = torch.zeros_like(scale).scatter_reduce_(
            0, ids.flatten()[:, None].expand(-1, scale.shape[1]), top, "amax") / most
        want = torch.where(held[:, None], torch.maximum(want, scale), want)
        want = torch.where(touched[:, None], want, scale)
        raw = _bytes(cache)
        # Earlier tokens of the first pages, in the page's new scale.
        codes = raw[first]
        old, now = scale[first][:, None, :, None], want[first][:, None, :, None]
        again = _bytes(_encode(codes.view(cache.dtype).float() * old, now, cache.dtype, most))
        change = (torch.arange(page, device=lens.device)[None] < before[:, None])[..., None, None]
        raw[first] = torch.where(change & (old != now), again, codes)
        raw[ids, slot] = _bytes(_encode(x, want[ids][..., None], cache.dtype, most))
        scale.copy_(want)
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _evict_plain(s):
    w, lens, page, budget = s["weights"], s["lens"].long(), s["page"], s["budget"]
    b, hkv, width = w.shape
    at = torch.arange(width, device=w.device)[None, None]
    n = lens[:, None, None]
    always = (at < s["sink"]) | (at >= n - s["recent"])
    rank = torch.where(at >= n, float("-inf"), torch.where(always, float("inf"), w))
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    best = best.sort(-1).values
    if best.shape[-1] < budget:  # a table of fewer tokens than the budget
        best = torch.cat([best, best.new_full((b, hkv, budget - best.shape[-1]), width - 1)], -1)
    new_lens = lens.clamp(max=budget)
    j = torch.arange(budget, device=w.device)
    real = (j[None] < new_lens[:, None])[:, None]
    kept = torch.where(real, best, -1)
    new_w = torch.where(real, w.gather(2, best), 0.0)
    # Past the kept tokens the last one again: the same write.
    last = (new_lens[:, None, None] - 1).expand(b, hkv, 1)
    best = torch.where(real, best, best.gather(2, last))
    to = torch.minimum(j[None], new_lens[:, None] - 1)  # [B, budget]
    heads = torch.arange(hkv, device=w.device)[None, :, None]
    from_page = s["tables"].long()[:, None].expand(-1, hkv, -1).gather(2, best // page)
    to_page = s["new_tables"].long().gather(1, to // page)[:, None].expand(-1, hkv, -1)
    to_slot = (to % page)[:, None]
    for cache, scale, new, new_scale in ((s["k"], s["k_scale"], s["new_k"], s["new_k_scale"]),
                                         (s["v"], s["v_scale"], s["new_v"], s["new_v_scale"])):
        x = _bytes(cache)[from_page, best % page, heads]
        if scale is not None:
            old = scale[from_page, heads]  # [B, Hkv, budget]
            blocks = -(-budget // page)
            pad = torch.zeros(b, hkv, blocks * page, device=w.device)
            pad[..., :budget] = torch.where(real, old, 0.0)
            block = pad.view(b, hkv, blocks, page).amax(-1)
            now = block.gather(2, (to // page)[:, None].expand(-1, hkv, -1))
            y = _bytes(_encode(x.view(cache.dtype).float() * old[..., None], now[..., None],
                               cache.dtype, s["code"]))
            x = torch.where((old != now)[..., None], y, x)
            new_scale[to_page, heads.expand_as(to_page)] = now
        _bytes(new)[to_page, to_slot.expand_as(to_page), heads.expand_as(to_page)] = x
    return (new_lens.to(torch.int32), new_w, kept.to(torch.int32), s["new_k"], s["new_v"],
            s["new_k_scale"], s["new_v_scale"])


OPERATORS = {"append": (_append_plain, _append_own), "attend": (_attend_plain, _attend_own),
             "weigh": (_weigh_plain, _weigh_own), "evict": (_evict_plain, _evict_own)}


def work(case):
    """Each input read once, each output written once."""
    lens = _lengths(case)
    es = 1 if case["kv"] in CODE_MAX else 2
    b, q, hq, hkv, d, page = (case[k] for k in ("batch", "q_len", "hq", "hkv", "d", "page"))
    token = hkv * d
    scales = 4 * hkv if es == 1 else 0  # of a page, for K or V
    tables = 4 * b + 4 * sum(-(-n // page) for n in lens)
    seen = sum(q * n - q * (q - 1) // 2 for n in lens)  # the draft chain
    if case["op"] == "append":
        n = sum(min(x, min(lens)) for x in _new(case))
        return {"bytes": 2 * n * token * (2 + es) + 2 * scales * n / page, "flops": 6 * n * token}
    if case["op"] == "attend":
        return {"bytes": 2 * (sum(lens) * token * es + scales * sum(lens) / page)
                + 4 * b * q * hq * d + tables, "flops": 4 * hq * d * seen}
    if case["op"] == "weigh":
        return {"bytes": sum(lens) * token * es + scales * sum(lens) / page + 2 * b * q * hq * d
                + 8 * hkv * sum(lens) + tables, "flops": 2 * hq * d * seen}
    kept = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": 4 * hkv * (sum(lens) + 2 * kept) + 2 * 2 * kept * token * es
            + 2 * 2 * scales * kept / page, "flops": 2 * sum(lens) * hkv}


# The definitions in 64 bits, sequence by sequence.

def _sequence(cache, scale, ids, n):
    """The first n tokens of one sequence, [Hkv, n, D]."""
    x = _bytes(cache)[ids].view(cache.dtype).double()
    if scale is not None:
        x *= scale[ids].double()[:, None, :, None]
    return x.flatten(0, 1)[:n].transpose(0, 1).contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    lens, page, op = s["lens"].tolist(), s["page"], s["op"]
    if op in ("attend", "weigh"):
        b, q_len, hq, d = s["query"].shape
        hkv = s["k"].shape[2]
        group = hq // hkv
        out = torch.zeros(b, q_len, hq, d, dtype=torch.float64, device="cuda")
        weights = s["weights"].double() if op == "weigh" else None
        for i, n in enumerate(lens):
            ids = s["tables"][i, :-(-n // page)].long()
            k = _sequence(s["k"], s["k_scale"], ids, n)
            seen = torch.ones(q_len, n, dtype=torch.bool, device="cuda")
            seen[:, n - q_len:] = (torch.ones_like(seen[:, :q_len]).tril() if s["trees"] is None
                                   else s["trees"][i])
            for h in range(hkv):
                for r in range(q_len):
                    q = s["query"][i, r, h * group:(h + 1) * group].double()
                    z = (q @ k[h].t()) / math.sqrt(d)
                    z[:, ~seen[r]] = float("-inf")
                    p = torch.softmax(z, -1)
                    if op == "weigh":
                        if r == 0:
                            weights[i, h, n - q_len:n] = 0
                        weights[i, h, :n] += p.sum(0)
                    else:
                        if r == 0 and h == 0:
                            v = _sequence(s["v"], s["v_scale"], ids, n)
                        out[i, r, h * group:(h + 1) * group] = p @ v[h]
        return weights if op == "weigh" else out
    if op == "append":
        got = []
        for x, cache, scale in ((s["key"], s["k"], s["k_scale"]),
                                (s["value"], s["v"], s["v_scale"])):
            # Codes unrounded: what the 8 bits stand for, in units of the page's scale.
            codes, scales = cache.double(), scale.double()
            for i, (n, m) in enumerate(zip(lens, s["new"].tolist())):
                for p in range((n - m) // page, -(-n // page)):
                    pid = int(s["tables"][i, p])
                    lo, hi = max(n - m, p * page), min(n, (p + 1) * page)
                    rows = x[i, lo - (n - m):hi - (n - m)].double()
                    now = rows.abs().amax((0, 2)) / s["code"]
                    if lo > p * page:
                        now = torch.maximum(now, scales[pid])
                        codes[pid, :lo - p * page] *= (scales[pid] / now)[:, None]
                    codes[pid, lo - p * page:hi - p * page] = rows / now[:, None]
                    scales[pid] = now
            got.append((codes, scales))
        return got[0][0], got[1][0], got[0][1], got[1][1]
    budget, sink, recent = s["budget"], s["sink"], s["recent"]
    w = s["weights"].double().cpu()
    b, hkv = w.shape[:2]
    new_w = torch.zeros(b, hkv, budget, dtype=torch.float64)
    new = [s[n].double() for n in ("new_k", "new_v")]
    new_scale = [x if x is None else x.double() for x in (s["new_k_scale"], s["new_v_scale"])]
    for i, n in enumerate(lens):
        ids = s["tables"][i, :-(-n // page)].long()
        m = min(n, budget)
        to = torch.arange(m, device="cuda")
        pid, slot = s["new_tables"][i].long()[to // page], to % page
        every = [_sequence(s[a], s[c], ids, n) for a, c in (("k", "k_scale"), ("v", "v_scale"))]
        for h in range(hkv):
            if n <= budget:
                keep = torch.arange(n)
            else:
                free = budget - sink - recent
                middle = w[i, h, sink:n - recent]
                order = sorted(range(len(middle)), key=middle.neg().tolist().__getitem__)[:free]
                keep = torch.cat([torch.arange(sink), torch.tensor(sorted(order)).long() + sink,
                                  torch.arange(n - recent, n)])
            new_w[i, h, :m] = w[i, h][keep]
            at = keep.cuda()
            for x, y, old, scale in zip(every, new, (s["k_scale"], s["v_scale"]), new_scale):
                if scale is None:
                    y[pid, slot, h] = x[h, at]
                    continue
                mine = old[ids[at // page], h].double()
                block = torch.zeros(-(-m // page), dtype=torch.float64, device="cuda")
                block = block.scatter_reduce_(0, to // page, mine, "amax")
                scale[s["new_tables"][i, :len(block)].long(), h] = block
                y[pid, slot, h] = x[h, at] / block[to // page][:, None]
    return (None, new_w.cuda(), None, new[0], new[1], new_scale[0], new_scale[1])
