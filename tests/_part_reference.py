"""Plain 64-bit statements of attention over a window and over a shared prefix, on the CPU,
and how far a kernel's result may be from them; inputs for both."""

from __future__ import annotations

import math

import torch

from tests._cache_reference import CODE_MAX, _product, half_step, quantise, tokens_of, visible

E4M3, INT8, F16, BF16 = torch.float8_e4m3fn, torch.int8, torch.float16, torch.bfloat16


def attention(q, k, v, k_scale, v_scale, tables, lens, seen_of, scale=None, out_scale=1.0,
              p_step=None):
    """``(out, bound)`` ``[B, Q, Hq, D]`` in 64 bits; ``seen_of(i, n)`` is the bool ``[Q, n]``
    of what the rows of sequence i see. Tokens nobody sees may be on no page at all.

    ``p_step``: how far a probability is from its rounding, relative to it. With 16-bit
    queries over caches without scales that is 2^-11 in fp16 (one rounding), 2^-17 in bf16
    (two parts of 8 bits); over codes with block scales 2^-11 for both."""
    b, q_len, hq, d = q.shape
    hkv = k.shape[2]
    group = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    if p_step is None:
        p_step = 2.0 ** -17 if q.dtype is BF16 and k_scale is None else 2.0 ** -11
    out = torch.zeros(b, q_len, hq, d, dtype=torch.float64)
    bound = torch.zeros_like(out)
    page = k.shape[1]
    for i, n in enumerate(int(x) for x in lens):
        if n <= 0:
            continue
        every = seen_of(i, n)
        at = every.any(0).nonzero()[:, 0]
        if len(at) == 0:
            continue
        seen, m = every[:, at], len(at)
        ids = tables[i].long()[at // page]
        assert (ids >= 0).all()

        def take(cache, s):
            raw = cache if cache.element_size() > 1 else cache.view(torch.uint8)
            x = raw[ids, at % page].contiguous().view(cache.dtype).double()
            return x if s is None else x * s[ids].double()[..., None]

        ks, vs = take(k, k_scale), take(v, v_scale)
        for h in range(hq):
            kk, vv, qq = ks[:, h // group], vs[:, h // group], q[i, :, h].double()
            s = qq @ kk.t() * scale
            # fp32 sums of d exact products, then the scale and the difference to the running
            # maximum: each a rounding of something no larger than `reach`.
            reach = torch.where(seen, qq.abs() @ kk.abs().t() * scale, 0.0).amax(1)
            delta = (d + 8) * reach * 2.0 ** -24 + 2.0 ** -20
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True)
            e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = e.sum(1, keepdim=True)
            p = torch.where(total == 0, 0.0, e / total)
            out[i, :, h] = out_scale * _special(p, vv, seen)
            size = abs(out_scale) * _product(p, vv.abs(), seen).nan_to_num(0.0, 0.0)
            # In units of the row's largest probability (times V scale), of which the row sum
            # is at least one, fp16 is off by 2^-25 where P is under 2^-14.
            big = torch.where(torch.isfinite(vv), vv.abs(), 0.0).amax()
            if v_scale is not None:
                big = CODE_MAX[v.dtype] * v_scale[ids, h // group].double().nan_to_num().max()
            tiny = m * 2.0 ** -25 * big if p_step == 2.0 ** -11 else 0.0
            # The probabilities in the product and in the row sum; fp32 sums; the scores in
            # both; the output's rounding, with its smallest step.
            bound[i, :, h] = size * (2 * p_step + m * 2.0 ** -23 + 2 * delta[:, None]) \
                + abs(out_scale) * tiny + half_step(q.dtype) * out[i, :, h].abs() * 1.01 + 2.0 ** -24
    return out, bound


def _special(p, v, seen):
    """``p @ v`` where tokens a row does not see take no part, whatever their values, and a
    value that is not finite counts as itself however small its probability."""
    out = p @ torch.where(torch.isfinite(v), v, 0.0)
    s = seen.double()
    up, down, nan = (s @ hit.double() > 0 for hit in (v == math.inf, v == -math.inf, v.isnan()))
    out = torch.where(up, math.inf, out)
    out = torch.where(down, -math.inf, out)
    return torch.where(nan | (up & down) | p.isnan().any(1, keepdim=True), math.nan, out)


def assert_within(actual, want, bound, label=""):
    """Every value within its bound, infinities and NaN where the definition has them."""
    a, w = actual.detach().double().cpu(), want.double()
    for what, test in (("NaN", torch.isnan), ("infinities", torch.isinf)):
        assert torch.equal(test(a), test(w)), f"{label}: {what} in other places"
    odd = ~torch.isfinite(w)
    assert torch.equal(torch.sign(a[torch.isinf(w)]), torch.sign(w[torch.isinf(w)])), label
    off = torch.where(odd, 0.0, (a - w).abs() - bound)
    if off.numel() and off.max() > 0:
        at = [int(x) for x in (off == off.max()).nonzero()[0]]
        raise AssertionError(f"{label}: {(off > 0).sum()} values off, worst at {at}: "
                             f"{a[tuple(at)]:.6g}, want {w[tuple(at)]:.6g} +- "
                             f"{bound[tuple(at)]:.3g}")


def window_seen(n, q_len, window, sink, tree=None):
    t = torch.arange(n)[None]
    p = n - q_len + torch.arange(q_len)[:, None]
    return visible(n, q_len, tree) & ((t < sink) | (t > p - window))


def cache(pool, page, hkv, d, dtype, kv, scaled, g, quiet=True):
    """One pool and its scales (None), values of ordinary size. With ``quiet`` False blocks
    differ by up to 2^12."""
    x = torch.randn(pool, page, hkv, d, generator=g)
    if scaled:
        if not quiet:
            x = x * 2.0 ** torch.randint(-8, 5, (pool, 1, hkv, 1), generator=g)
        return quantise(x, kv)
    return x.to(kv or dtype), None


def spoil(codes, ids, slots=None):
    """NaN (e4m3, 16-bit) or the lowest integer into pages ``ids`` or their ``slots``."""
    raw = codes.view(torch.uint8) if codes.element_size() == 1 else codes
    junk = {E4M3: 0x7F, INT8: 0x80}.get(codes.dtype, float("nan"))
    if slots is None:
        raw[ids] = junk
    else:
        raw[ids, slots] = junk


def trees(b, q_len, seed=0, empty=()):
    """Random draft trees; rows in ``empty`` see no draft token."""
    g = torch.Generator().manual_seed(seed)
    seen = torch.rand(b, q_len, q_len, generator=g) < 0.5
    for r in empty:
        if r < q_len:
            seen[:, r] = False
    return seen


def window_inputs(lens, q_len, hq, hkv, d, page, dtype, kv, scaled, window, sink, seed=0,
                  width=None, quiet=True):
    """Query, caches, scales, tables, lengths on the CPU. Pages of tokens that no row's
    window reaches are on no page (-1); tokens nobody sees, pages nobody owns and slots past
    the end hold NaN."""
    g = torch.Generator().manual_seed(seed)
    live = []
    for n in lens:
        n = max(n, 0)
        t = torch.arange(n)
        seen = (t < sink) | (t >= n - q_len + 1 - window)
        live.append(sorted(set((t[seen] // page).tolist())))
    pool = sum(len(x) for x in live) + 3
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    most = max([-(-max(n, 0) // page) for n in lens] + [1])
    tables = torch.full((len(lens), width or most), -1, dtype=torch.int32)
    at = 0
    for i, pages in enumerate(live):
        tables[i, pages] = perm[at:at + len(pages)]
        at += len(pages)
    q = torch.randn(len(lens), q_len, hq, d, generator=g).to(dtype)
    caches, scales = zip(*(cache(pool, page, hkv, d, dtype, kv, scaled, g, quiet)
                           for _ in range(2)))
    for c, s in zip(caches, scales):
        spoil(c, perm[at:].long())
        if s is not None:
            s[perm[at:].long()] = float("nan")
        for i, n in enumerate(lens):
            for pg in live[i]:
                t = pg * page + torch.arange(page)
                dead = (t >= n) | ((t >= sink) & (t < n - q_len + 1 - window))
                if dead.any():
                    spoil(c, int(tables[i, pg]), dead.nonzero()[:, 0])
    return q, list(caches), list(scales), tables, torch.tensor(lens, dtype=torch.int32)


def cuda(*xs):
    return [None if x is None else x.cuda() for x in xs]


__all__ = ["attention", "assert_within", "window_seen", "window_inputs", "trees", "cuda", "cache",
           "spoil", "tokens_of"]
