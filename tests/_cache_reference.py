"""Plain 64-bit statements of the operators around the paged cache, on the CPU, and how
far a kernel's result may be from them.

Each is written from the operator's definition alone, sequence by sequence."""

from __future__ import annotations

import math

import torch

CODE_MAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def half_step(dtype) -> float:
    """Relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def quantise(x, dtype):
    """``[P, page, Hkv, D]`` values -> codes and ``[P, Hkv]`` scales (a cache to read)."""
    most = CODE_MAX[dtype]
    scale = (x.abs().amax((1, 3)) / most).float()
    y = torch.where(scale[:, None, :, None] > 0, x / scale[:, None, :, None], 0.0)
    y = (y.round() if dtype is torch.int8 else y).clamp(-most, most)
    return y.to(dtype), scale


def tokens_of(cache, scale, table, n):
    """The first ``n`` tokens of a sequence in 64 bits, ``[n, Hkv, D]``."""
    page = cache.shape[1]
    ids = table[:-(-n // page)].long()
    raw = cache if cache.element_size() > 1 else cache.view(torch.uint8)
    x = raw[ids].contiguous().view(cache.dtype).double()
    if scale is not None:
        x = x * scale[ids].double()[:, None, :, None]
    return x.flatten(0, 1)[:n]


def visible(n, q_len, tree):
    """``[Q, n]``: which tokens draft row i sees (``tree``: bool ``[Q, Q]`` or None)."""
    t = torch.arange(n)[None]
    i = torch.arange(q_len)[:, None]
    if tree is None:
        return t < n - q_len + i + 1
    j = t - (n - q_len)
    at = j.clamp(0, q_len - 1).expand(q_len, n)
    return (j < 0) | tree.gather(1, at)


def attention(q, k, v, k_scale, v_scale, tables, lens, trees=None, scale=None, out_scale=1.0):
    """``(out, bound, probabilities)`` in 64 bits: ``out`` ``[B, Q, Hq, D]``, ``bound`` the
    error that roundings may leave in it, ``probabilities`` per sequence ``[Hkv, Q, n]``
    summed over a head group's query heads, with their bound."""
    b, q_len, hq, d = q.shape
    hkv = k.shape[2]
    group = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, q_len, hq, d, dtype=torch.float64)
    bound = torch.zeros_like(out)
    mass = []
    for i, n in enumerate(int(x) for x in lens):
        weights = torch.zeros(hkv, q_len, max(n, 0), dtype=torch.float64)
        far = torch.zeros_like(weights)
        mass.append((weights, far))
        if n <= 0:
            continue
        ks = tokens_of(k, k_scale, tables[i], n)
        vs = tokens_of(v, v_scale, tables[i], n) if v is not None else None
        seen = visible(n, q_len, None if trees is None else trees[i])
        for h in range(hq):
            kk = ks[:, h // group]
            qq = q[i, :, h].double()
            s = qq @ kk.t() * scale
            # fp32 sums of d exact products, then the scale and the difference to the
            # running maximum: each a rounding of something no larger than `reach`.
            reach = (qq.abs() @ kk.abs().t() * scale)
            reach = torch.where(seen, reach, 0.0).amax(1)
            delta = (d + 8) * reach * 2.0 ** -24 + 2.0 ** -20
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True)
            e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = e.sum(1, keepdim=True)
            p = torch.where(total == 0, 0.0, e / total)
            weights[h // group] += p
            far[h // group] += p * (2 * delta[:, None] + n * 2.0 ** -24)
            if vs is None:
                continue
            vv = vs[:, h // group]
            out[i, :, h] = out_scale * _product(p, vv, seen)
            size = abs(out_scale) * _product(p, vv.abs(), seen)
            # P = p v_scale, rounded once to fp16 for the product with the codes: off by
            # 2^-11 of itself, or, below 2^-14, by 2^-25. It is taken relative to a maximum
            # no larger than the row's largest p v_scale, call it p* s*: in those units the
            # row sum is at least 1 / s*, so the n roundings of 2^-25, each times a code,
            # leave at most n 2^-25 (largest code) s* in the quotient. Then fp32 sums, the
            # scores' errors (twice: numerator and denominator), the output's rounding.
            loudest = vs.new_zeros(())
            if v_scale is not None:
                pages = tables[i, :-(-n // v.shape[1])].long()
                loudest = CODE_MAX[v.dtype] * v_scale[pages, h // group].double().nan_to_num().max()
            bound[i, :, h] = size * (2.0 ** -11 + n * 2.0 ** -23 + 2 * delta[:, None]) \
                + abs(out_scale) * n * 2.0 ** -25 * loudest \
                + half_step(q.dtype) * out[i, :, h].abs() * 1.01 + 2.0 ** -24
    return out, bound, mass


def _product(p, v, seen):
    """``p @ v`` where tokens a row does not see take no part, whatever their values."""
    clean = p @ torch.where(torch.isfinite(v), v, 0.0)
    hit = seen.double() @ (~torch.isfinite(v)).double()
    return torch.where(hit > 0, math.nan, clean)


def assert_within(actual, want, bound, label=""):
    """Every value within its bound, NaN where the definition gives NaN."""
    a, w = actual.detach().double().cpu(), want.double()
    nan = torch.isnan(w)
    assert torch.equal(torch.isnan(a), nan), f"{label}: NaN in other places"
    off = torch.where(nan, 0.0, (a - w).abs() - bound)
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0, f"{label}: {worst:.3g} past the bound (largest difference " \
        f"{torch.where(nan, 0.0, (a - w).abs()).max().item():.3g})"


def append(key, value, caches, scales, tables, lens, new_lens=None):
    """The quantising append on CPU tensors, in place; the new scales in 32 bits (they are
    part of the result), the codes rounded from 64 bits. ``ties`` of the returned dict:
    codes whose quotient lies so near a border that 32-bit division may round it the
    other way."""
    page, dtype = caches[0].shape[1], caches[0].dtype
    most = CODE_MAX[dtype]
    ties = [torch.zeros(c.shape, dtype=torch.bool) for c in caches]
    for x, cache, scale, tie in zip((key, value), caches, scales, ties):
        raw = cache.view(torch.uint8)
        top = torch.finfo(x.dtype).max
        for i, n in enumerate(int(v) for v in lens):
            n = max(n, 0)
            m = x.shape[1] if new_lens is None else int(new_lens[i])
            m = max(0, min(m, x.shape[1], n))
            if m == 0:
                continue
            for p in range((n - m) // page, -(-n // page)):
                if p >= tables.shape[1] or not 0 <= int(tables[i, p]) < cache.shape[0]:
                    continue
                pid = int(tables[i, p])
                lo, hi = max(n - m, p * page), min(n, (p + 1) * page)
                a, z = lo - p * page, hi - p * page
                rows = x[i, lo - (n - m):hi - (n - m)].double().clamp(-top, top)
                now = (torch.nan_to_num(rows, nan=0.0).abs().amax((0, 2)).float() / most)
                old = scale[pid].clone()
                if a > 0:
                    now = torch.maximum(now, old)
                    kept = cache[pid, :a].double() * (old.double() / now.double())[:, None]
                    grown = (now != old)[:, None].expand(kept.shape[1:])
                    codes, near = _encode(kept, dtype, most)
                    raw[pid, :a] = torch.where(grown, codes, raw[pid, :a])
                    tie[pid, :a] = near & grown
                codes, near = _encode(torch.where(now[:, None] > 0, rows / now.double()[:, None],
                                                  0.0), dtype, most)
                raw[pid, a:z] = codes
                tie[pid, a:z] = near
                scale[pid] = now
    return ties


def _encode(y, dtype, most):
    """Codes as bytes, and where 32-bit arithmetic may end on the other side of a border."""
    def code(v):
        v = v.clamp(-most, most)
        if dtype is torch.int8:
            return torch.nan_to_num(v, nan=0.0).round().to(torch.int8).view(torch.uint8)
        # float64 -> e4m3 in one rounding: float32 holds e4m3's borders exactly, so a
        # value pushed onto one by the first rounding is a tie that is reported.
        return v.float().to(torch.float8_e4m3fn).view(torch.uint8)

    # Products and quotients of 32-bit values: within three roundings.
    near = code(y * (1 + 2.0 ** -22)) != code(y * (1 - 2.0 ** -22))
    return code(y), near


def weights_after(old, mass, lens, q_len):
    """``(weights, bound)`` after a call whose probabilities are ``mass`` (:func:`attention`)."""
    want = old.double().clone()
    bound = torch.zeros_like(want)
    width = old.shape[2]
    for i, n in enumerate(max(int(x), 0) for x in lens):
        p, far = (x.sum(1)[:, :width] for x in mass[i])
        draft = max(n - q_len, 0)
        want[i, :, draft:n] = 0.0
        want[i, :, :n] += p
        # The rows' sum and the addition to the old value, in 32 bits.
        bound[i, :, :n] = far + 80 * 2.0 ** -24 * p + 2.0 ** -24 * want[i, :, :n].abs() + 1e-30
    return want, bound


def kept_tokens(weights, n, budget, sink, recent):
    """Positions that stay of a sequence of ``n`` tokens with these weights (a list)."""
    if n <= budget:
        return list(range(n))
    middle = range(sink, n - recent)
    w = [float(x) for x in weights]
    order = sorted(middle, key=lambda t: (math.isnan(w[t]), -w[t] if w[t] == w[t] else 0.0, t))
    chosen = order[:budget - sink - recent]
    return sorted(list(range(sink)) + chosen + list(range(n - recent, n)))


def evict(weights, caches, scales, tables, lens, new_tables, budget, sink, recent, into,
          into_scales):
    """Eviction on CPU tensors: moves into ``into`` (and ``into_scales``) and returns
    ``(new_lens, new_weights, kept)``."""
    b, hkv, _ = weights.shape
    page = caches[0].shape[1]
    kept = torch.full((b, hkv, budget), -1, dtype=torch.int32)
    new_w = torch.zeros(b, hkv, budget)
    new_lens = torch.clamp(lens, min=0).clamp(max=budget)
    for i in range(b):
        n = max(int(lens[i]), 0)
        for h in range(hkv):
            stay = kept_tokens(weights[i, h], n, budget, sink, recent)
            kept[i, h, :len(stay)] = torch.tensor(stay, dtype=torch.int32)
            new_w[i, h, :len(stay)] = weights[i, h, stay]
            for which in range(2):
                cache, new = caches[which], into[which]
                raw = cache.view(torch.uint8) if cache.element_size() == 1 else cache
                raw_new = new.view(torch.uint8) if new.element_size() == 1 else new
                for p in range(-(-len(stay) // page)):
                    to = int(new_tables[i, p])
                    part = stay[p * page:(p + 1) * page]
                    from_pages = [int(tables[i, t // page]) for t in part]
                    if scales is not None:
                        now = max(scales[which][f, h] for f in from_pages)
                        into_scales[which][to, h] = now
                    for slot, (t, f) in enumerate(zip(part, from_pages)):
                        x = raw[f, t % page, h]
                        if scales is not None and scales[which][f, h] != now:
                            # In 32 bits, operation by operation: part of the definition.
                            y = cache[f, t % page, h].float() * scales[which][f, h] / now
                            y = (y.round() if cache.dtype is torch.int8 else y)
                            x = y.clamp(-CODE_MAX[cache.dtype], CODE_MAX[cache.dtype]) \
                                .to(cache.dtype).view(torch.uint8)
                        raw_new[to, slot, h] = x
    return new_lens, new_w, kept
