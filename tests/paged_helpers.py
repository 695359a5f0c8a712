"""Oracles of the 8-bit paged cache and its attention in 64 bits (torch, any
device), and the inputs of their tests."""

from __future__ import annotations

import math

import torch

F8 = torch.float8_e4m3fn
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


def e4m3_table():
    """The 256 code values in f64, from the format's definition: sign, 4 exponent
    bits biased by 7, 3 mantissa bits; 0x7f / 0xff are NaN."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        out.append(math.nan if c & 127 == 127 else (-v if c & 128 else v))
    return torch.tensor(out, dtype=torch.float64)


def nearest_codes(x):
    """Code of each x (f64): the nearest value, ties to the even code, at most
    448; 0x7f for what is not finite.  By search among the code values."""
    vals = e4m3_table()[:127].to(x.device)  # increasing
    a = x.abs().clamp(max=448.0)
    hi = torch.searchsorted(vals, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - vals[lo], vals[hi] - a
    code = torch.where(dl < dh, lo, torch.where(dh < dl, hi, torch.where(lo % 2 == 0, lo, hi)))
    code = torch.where(a == vals[hi], hi, code)
    code = code + 128 * torch.signbit(x).long()
    return torch.where(x.isfinite(), code, 0x7f).to(torch.uint8)


def row_bytes(x):
    """E8M0 byte of each row of x (f64): the smallest e in [1, 254] with
    max |x| <= 448 * 2^(e - 127) over the finite elements, by trying them all."""
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    s = 448.0 * torch.exp2(torch.arange(1, 255, dtype=torch.float64, device=x.device) - 127)
    return (torch.searchsorted(s, amax.contiguous()) + 1).clamp(max=254).to(torch.uint8)


def quantise(x, scaled, factor=1.0):
    """(codes, bytes or None) of rows x."""
    if not scaled:
        # (the quotient is an IEEE fp32 division: its rounding is part of the format;
        # one of a finite x that overflows saturates)
        y = (x.float() / torch.tensor(factor, dtype=torch.float32, device=x.device)).double()
        return nearest_codes(torch.where(x.isfinite(), y.clamp(-448.0, 448.0), y)), None
    b = row_bytes(x.double())
    return nearest_codes(x.double() * torch.exp2(127 - b.double())[..., None]), b


def values(codes, byte, factor):
    """f64 values of rows of codes (uint8)."""
    x = e4m3_table().to(codes.device)[codes.long()]
    return x * torch.exp2(byte.double() - 127)[..., None] if byte is not None else x * factor


def make_cache(gen, pages, page, hkv, d, kind, dtype, device, layout="nhd"):
    """(k_cache, v_cache, kv_scales, k_scale, v_scale, k f64, v f64): a cache of
    random rows, kind "fp8", "static" or "same"; the f64 rows [pages * page, Hkv, D]
    are the values it holds."""
    n = pages * page
    rows = [torch.randn(n, hkv, d, generator=gen, device=device) * torch.exp2(torch.randn(n, hkv, 1, generator=gen, device=device))
            for _ in range(2)]
    ks = vs = 1.0
    sc, caches, vals = None, [], []
    if kind == "static":
        ks, vs = 0.03125, 0.021
    if kind == "fp8":
        sc = torch.zeros(pages, hkv, page, 2, dtype=torch.uint8, device=device)
    for i, (x, f) in enumerate(zip(rows, (ks, vs))):
        if kind == "same":
            c = x.to(dtype).view(pages, page, hkv, d)
            vals.append(c.double().reshape(n, hkv, d))
        else:
            code, byte = quantise(x, kind == "fp8", f)
            vals.append(values(code, byte, float(torch.tensor(f, dtype=torch.float32))))
            c = code.view(F8).view(pages, page, hkv, d)
            if byte is not None:
                sc[..., i] = byte.view(pages, page, hkv).transpose(1, 2)
        caches.append(c)
    if layout == "hnd":  # pages of [Hkv, page, D]
        caches = [_u8(c).transpose(1, 2).contiguous().transpose(1, 2).view(c.dtype) for c in caches]
    elif layout == "interleaved":  # K and V pages after one another
        both = torch.stack([_u8(c) for c in caches], 1).contiguous()
        caches = [both[:, i].view(c.dtype) for i, c in enumerate(caches)]
    return caches[0], caches[1], sc, ks, vs, vals[0], vals[1]


def _u8(c):
    return c.view(torch.uint8) if c.dtype == F8 else c


def attention(q, k, v, new, lens, table, page, num_pages, sm, window=-1, cap=0.0, req_ids=None):
    """(out, lse, tol_out, tol_lse) f64 of requests whose rows follow one another.

    Tolerances.  With u half a step of q's type: the output is rounded once (u
    |out|), and every weight is rounded to that type for its product (u of it,
    so u A with A = sum p |v| / l).  A score is an fp32 sum of D products (|ds| <=
    D 2^-24 sum |q k| sm, 2^-24 |s| for the scale's fma; with a cap the capped
    score, 2^-20 cap for tanh), which moves lse by as much and each weight by
    twice that (its own and the sum's); exp2, log2 and the fp32 sums add 2^-18
    (hardware exp2 and log2 to 1 ulp; l sums n terms in at most n/32/4 + 8
    sequential steps, each 2^-24, of positive terms: below 2^-14 for the sizes
    here, which `steps` counts)."""
    hq, d = q.shape[1], q.shape[2]
    g = hq // k.shape[1]
    u = U[q.dtype]
    outs, lses, touts, tlses = [], [], [], []
    at = 0
    for b, (n, ln) in enumerate(zip(new, lens)):
        row = b if req_ids is None else req_ids[b]
        cap_keys = table.shape[1] * page if 0 <= row < table.shape[0] else 0
        nk = min(max(ln, 0), cap_keys)
        key = torch.arange(nk, device=q.device)
        ent = table[row].long()[key // page] if nk else key
        ok = (ent >= 0) & (ent < num_pages)
        slot = torch.where(ok, ent, 0) * page + key % page
        pos = max(ln, 0) - n + torch.arange(n, device=q.device)[:, None]
        seen = (key <= pos) & ok
        if window >= 0:
            seen = seen & (key >= pos - window)
        kk, vv = k[slot], v[slot]
        for h in range(hq):
            qq = q[at:at + n, h].double()
            w = qq @ kk[:, h // g].T.contiguous() * sm
            mag = qq.abs() @ kk[:, h // g].abs().T.contiguous() * sm
            mag = torch.where(seen, mag, 0.0).amax(1) if nk else torch.zeros(n, device=q.device, dtype=torch.float64)
            if cap:
                w = cap * torch.tanh(w / cap)
            w = torch.where(seen, w, -math.inf)
            lse = torch.logsumexp(w, 1) if nk else torch.full((n,), -math.inf, device=q.device, dtype=torch.float64)
            p = torch.exp(w - torch.where(lse.isfinite(), lse, 0.0)[:, None])
            vm = torch.where(seen.any(0)[:, None], vv[:, h // g], 0.0) if nk else vv[:, h // g]
            o = p @ vm
            a = p @ vm.abs()
            steps = nk * 2.0 ** -24 / 32 + 2.0 ** -18
            tl = (d + 4) * 2.0 ** -24 * mag + (2.0 ** -20 * cap) + steps * (1 + lse.abs().nan_to_num(posinf=0.0))
            outs.append((at, h, o))
            lses.append((at, h, lse))
            touts.append(u * o.abs() + ((u + 2 * tl + steps)[:, None] * a) * 1.01 + 1e-30)
            tlses.append(tl)
        at += n
    total = at
    out = torch.zeros(total, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.zeros(total, hq, dtype=torch.float64, device=q.device)
    to, tl = torch.zeros_like(out), torch.zeros_like(lse)
    for (at, h, o), (_, _, s), a, c in zip(outs, lses, touts, tlses):
        out[at:at + o.shape[0], h] = o
        lse[at:at + o.shape[0], h] = s
        to[at:at + o.shape[0], h] = a
        tl[at:at + o.shape[0], h] = c
    return out, lse, to, tl


def offsets(new):
    qo = [0]
    for n in new:
        qo.append(qo[-1] + n)
    return qo


def page_table(gen, lens, page, device, extra=1, pages=None):
    """Scattered pages for every request; (table, number of pages)."""
    need = [-(-max(n, 0) // page) for n in lens]
    pages = pages or sum(need) + 2
    order = torch.randperm(pages, generator=gen, device=device).int()
    table = torch.full((len(lens), max(need + [0]) + extra), -1, dtype=torch.int32, device=device)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def assert_close(got, want, tol, what):
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol))
    if bad.any():
        i = bad.nonzero()[0].tolist()
        worst = ((got - want).abs() / tol)[bad & want.isfinite()]
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at {i}: {float(got[tuple(i)])!r}, want "
                             f"{float(want[tuple(i)])!r} +- {float(tol[tuple(i)]):.3g}; worst {float(worst.max()) if worst.numel() else 0:.3g} tol")
