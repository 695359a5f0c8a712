"""Serving over an 8-bit paged K/V cache: the operators as cases to measure.

Four operators, each through the public entry points of the SGLang binding
(``load_mac_paged_cache_extension``):

* ``write``: the K and V rows of a chunk (or of a decode batch) quantised to
  e4m3 as they are written into their pages.
* ``rope``: a decode batch's RoPE, with the rotated keys and the values
  quantised into the cache by the same call.
* ``read``: cached rows of an index list read back as 16- or 32-bit rows.
* ``attn``: attention of a chunk of new tokens (one: a decode step; a few: the
  drafts of a speculative step; many: chunked prefill) over a paged cache of
  8- or 16-bit rows.

The cache: e4m3 K and V pages [pages, P, Hkv, D] and, in the row-scaled form,
one scale per row of K and of V in kv_scales [pages, Hkv, P, 2], an E8M0 byte e
for 2^(e - 127): the smallest power of two s with max |x| <= 448 s over the
row's finite elements.  The static form has one factor for K and one for V.

``run`` computes the plain forms in elementary torch operations while ``own``
is False, and calls the framework's kernels where it is True.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
STATIC_K, STATIC_V = 0.03125, 0.021  # calibrated factors of a static cache
POSITIONS = 131072


# ------------------------------------------------------------------ cases ---


def _write(name, tokens, hkv, d, page, dtype="bf16", scaled=True, fused_qkv=True):
    c = dict(op="write", tokens=tokens, hkv=hkv, d=d, page=page, dtype=dtype, scaled=scaled, fused_qkv=fused_qkv)
    return dict(c, name=name) if name else c


def _rope(name, tokens, hq, hkv, d, rot, page, dtype="bf16", neox=True, scaled=True):
    c = dict(op="rope", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, page=page, dtype=dtype, neox=neox, scaled=scaled)
    return dict(c, name=name) if name else c


def _read(name, tokens, hkv, d, page, dtype="bf16", scaled=True):
    c = dict(op="read", tokens=tokens, hkv=hkv, d=d, page=page, dtype=dtype, scaled=scaled)
    return dict(c, name=name) if name else c


def _attn(name, batch, rows, kv, hq, hkv, d, page, dtype="bf16", cache="fp8", ragged=False, window=-1, cap=0.0):
    """``rows`` new tokens per request over ``kv`` keys (the new ones among
    them); ragged: up to so many, each request with its own."""
    c = dict(op="attn", batch=batch, rows=rows, kv=kv, hq=hq, hkv=hkv, d=d, page=page, dtype=dtype, cache=cache,
             ragged=ragged, window=window, cap=cap)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the K/V write of a decode batch, K and V as views of the fused qkv rows
        _write("write_decode_b64", 64, 8, 128, 16),
        # the write of a server's largest prefill chunks
        _write("write_chunk_32768", 32768, 8, 128, 16),
        # decode RoPE with the write, token-indexed pool (page size 1)
        _rope("rope_decode_b64", 64, 32, 8, 128, 128, 1),
        # the same for a small prefill chunk, half-rotated heads in adjacent pairs
        _rope("rope_chunk_2048", 2048, 32, 8, 128, 64, 16, dtype="f16", neox=False),
        # a few hundred rows of a statically scaled cache read back
        _read("read_static_777", 777, 4, 64, 32, dtype="f16", scaled=False),
        # a long prefix read back for a kernel that wants 16-bit rows
        _read("read_prefix_65536", 65536, 8, 128, 16),
        # one request's decode step at a short context, token-indexed pool:
        # the smallest call
        _attn("attn_decode_b1_4k", 1, 1, 4096, 32, 8, 128, 1),
        # a full decode batch at long, unequal contexts: the step that the
        # cache's bytes bound
        _attn("attn_decode_b64_64k", 64, 1, 65536, 32, 8, 128, 16, ragged=True),
        # five drafted tokens a request over a 16-bit cache, 8 heads per KV head
        _attn("attn_draft_b32_16k", 32, 5, 16384, 32, 4, 128, 1, cache="same"),
        # a prefill chunk over a long prefix: the matrix cores' case
        _attn("attn_chunk_8192_32k", 1, 8192, 32768, 32, 8, 128, 16),
        # windowed layers with large heads and a logit cap, ragged chunks
        _attn("attn_window_d256_cap", 8, 1024, 8192, 16, 8, 256, 64, window=4095, ragged=True, cap=50.0),
        # a mixed batch (decode rows and small chunks), small heads, fp16, no
        # shared KV heads
        _attn("attn_mixed_b24_d64_f16", 24, 384, 6000, 16, 16, 64, 32, dtype="f16", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["write", "rope", "read", "attn", "attn", "attn", "attn", "attn"])
    hkv, d, page = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 128, 128, 256]), rng.choice([1, 1, 16, 16, 32, 64])
    dtype, scaled = rng.choice(["bf16", "bf16", "f16"]), rng.random() < 0.75
    most = 32768 * 8 * 128  # elements of K that the largest listed write has
    if op == "write":
        return _write(None, _log(rng, 1, most // (hkv * d)), hkv, d, page, dtype, scaled, rng.random() < 0.7)
    if op == "rope":
        g = rng.choice([1, 2, 4, 4, 7, 8])
        return _rope(None, _log(rng, 1, most // (hkv * d * (g + 2))), g * hkv, hkv, d, rng.choice([d, d, d // 2]), page,
                     dtype, rng.random() < 0.7, scaled)
    if op == "read":
        return _read(None, _log(rng, 1, 2 * most // (hkv * d)), hkv, d, page, rng.choice(["bf16", "bf16", "f16", "f32"]),
                     scaled)
    cache = rng.choice(["fp8", "fp8", "fp8", "static", "same"])
    g = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    kind = rng.choice(["decode", "decode", "draft", "chunk", "chunk"])
    if kind == "decode":
        batch, rows = _log(rng, 1, 128), 1
    elif kind == "draft":
        batch, rows = _log(rng, 1, 64), rng.randrange(2, 17)
    else:
        batch, rows = _log(rng, 1, 16), _log(rng, 17, 4096)
    width = 2 if cache == "same" else 1
    # at most the bytes of the largest listed decode step, the operations of
    # the largest listed chunk, and its padded score matrix
    top = min(POSITIONS, 3_600_000_000 // (batch * hkv * d * 2 * width), 3_000_000_000_000 // (4 * d * g * hkv * rows * batch),
              6_000_000_000 // (batch * hkv * g * rows))
    kv = max(rows, _log(rng, 1 if rng.random() < 0.2 else 200, max(top, 256)))
    window = -1 if rng.random() < 0.7 else _log(rng, 16, 4096)
    return _attn(None, batch, rows, kv, g * hkv, hkv, d, page, dtype, cache, rng.random() < 0.7, window,
                 rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]))


def _lengths(case):
    """(new tokens, keys) of every request: the case's own, whatever the seed."""
    n, rows, kv = case["batch"], case["rows"], case["kv"]
    if not case["ragged"]:
        return [rows] * n, [kv] * n
    rng = random.Random(",".join(f"{k}={case[k]}" for k in sorted(case) if k != "name"))
    new = [rows] + [_log(rng, 1, rows) for _ in range(n - 1)]
    keys = [kv] + [max(r, _log(rng, max(kv // 8, 1), kv)) for r in new[1:]]
    at = rng.randrange(n)  # the longest request is not always the first
    new[0], new[at], keys[0], keys[at] = new[at], new[0], keys[at], keys[0]
    return new, keys


# ------------------------------------------------------------ the format ---


def _row_scale(x):
    """E8M0 bytes of rows x (f32): the smallest power of two s with
    max |x| <= 448 s over the finite elements."""
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    return (e + 127 - 9 + (m > 0.875)).clamp(1, 254).to(torch.uint8)


def _power(byte):
    """2^(byte - 127) in f32."""
    return torch.ldexp(torch.ones((), device=byte.device), byte.to(torch.int32) - 127)


def _codes(x):
    """e4m3 of x (f32): the nearest, ties to even, at most 448; NaN for NaN and
    infinities."""
    return torch.where(x.isfinite(), x.clamp(-448.0, 448.0), math.nan).to(F8)


def _quantise(x, scaled, factor):
    """Codes and row bytes (None in the static form) of rows x."""
    x = x.float()
    if not scaled:
        return _codes(x / factor), None
    byte = _row_scale(x)
    return _codes(x * _power(254 - byte)[..., None]), byte


def _bits(t):
    return t.view(torch.uint8)


# --------------------------------------------------------------- prepare ---


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _rows(g, n, heads, d, dtype):
    """Rows of N(0, 1) times the row's own magnitude: tokens differ in size."""
    x = torch.empty(n, heads, d, device=DEV, dtype=torch.float32).normal_(generator=g)
    return x.mul_(torch.exp2(torch.empty(n, heads, 1, device=DEV).normal_(generator=g) * 0.7)).to(TYPES[dtype])


def _pool(g, pages, page, hkv, d, scaled):
    """A cache in use: K and V codes and the row scales."""
    n = pages * page
    kc, vc = (torch.empty(pages, page, hkv, d, device=DEV, dtype=F8) for _ in range(2))
    sc = torch.empty(pages, hkv, page, 2, device=DEV, dtype=torch.uint8) if scaled else None
    step = max(page, (1 << 26) // (hkv * d) // page * page)  # (slices: the 32-bit rows are 4 times the codes)
    for at in range(0, n, step):
        m = min(step, n - at)
        for i, (c, f) in enumerate(((kc, STATIC_K), (vc, STATIC_V))):
            code, byte = _quantise(_rows(g, m, hkv, d, "f32"), scaled, f)
            _bits(c)[at // page:(at + m) // page] = _bits(code).view(m // page, page, hkv, d)
            if scaled:
                sc[at // page:(at + m) // page, :, :, i] = byte.view(m // page, page, hkv).transpose(1, 2)
    return kc, vc, sc


def _i32(xs):
    return torch.tensor(xs, device=DEV, dtype=torch.int32)


def _ext():
    """The framework's operators (own form only)."""
    import os
    import sys

    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mac-attention_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mac_attention.integrations.sglang import bridge

    return bridge.load_mac_paged_cache_extension(False)


def _prepare_attn(case, seed):
    g = _gen(seed)
    new, keys = _lengths(case)
    b, hq, hkv, d, page = case["batch"], case["hq"], case["hkv"], case["d"], case["page"]
    need = [-(-k // page) for k in keys]
    pages = sum(need) + 3
    if case["cache"] == "same":
        kc, vc = (torch.empty(pages, page, hkv, d, device=DEV, dtype=TYPES[case["dtype"]]).normal_(generator=g)
                  for _ in range(2))
        sc = None
    else:
        kc, vc, sc = _pool(g, pages, page, hkv, d, case["cache"] == "fp8")
    order = torch.randperm(pages, generator=g, device=DEV).int()  # pages scattered over the pool
    table = torch.full((b, max(need)), -1, device=DEV, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    qo = [0]
    for n in new:
        qo.append(qo[-1] + n)
    return dict(q=_rows(g, qo[-1], hq, d, case["dtype"]), kc=kc, vc=vc, sc=sc, table=table, qo=_i32(qo), lens=_i32(keys),
                most=(max(new), max(keys)), ks=STATIC_K if case["cache"] == "static" else 1.0,
                vs=STATIC_V if case["cache"] == "static" else 1.0, sm=1.0 / math.sqrt(d))


def prepare(case, seed):
    op = case["op"]
    if op == "attn":
        s = _prepare_attn(case, seed)
    else:
        g = _gen(seed)
        n, hkv, d, page = case["tokens"], case["hkv"], case["d"], case["page"]
        pages = -(-n // page) + 5
        kc, vc, sc = _pool(g, pages, page, hkv, d, case["scaled"])
        it = torch.int64 if n % 2 else torch.int32
        loc = torch.randperm(pages * page, generator=g, device=DEV)[:n].to(it)
        s = dict(kc=kc, vc=vc, sc=sc, loc=loc, ks=1.0 if case["scaled"] else STATIC_K,
                 vs=1.0 if case["scaled"] else STATIC_V)
        if op == "write" and not case["fused_qkv"]:
            s.update(k=_rows(g, n, hkv, d, case["dtype"]), v=_rows(g, n, hkv, d, case["dtype"]))
        elif op != "read":  # views of the projection's fused rows
            hq = case.get("hq", 4 * hkv)
            q, k, v = _rows(g, n, hq + 2 * hkv, d, case["dtype"]).split([hq, hkv, hkv], dim=1)
            s.update(q=q, k=k, v=v)
        if op == "rope":
            rot = case["rot"]
            inv = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
            angle = torch.arange(POSITIONS, device=DEV, dtype=torch.float64)[:, None] * inv
            s.update(cs=torch.cat([angle.cos(), angle.sin()], 1).float(),
                     pos=torch.randint(0, POSITIONS, (n,), generator=g, device=DEV).to(it))
    return dict(s, case=case)


# ------------------------------------------------------------ plain forms ---


def _store(cache, sc, i, page, loc, code, byte):
    _bits(cache)[loc // page, loc % page] = _bits(code)
    if sc is not None:
        sc[loc // page, :, loc % page, i] = byte


def _plain_write(s, k, v):
    c = s["case"]
    loc = s["loc"].long()
    for i, (x, cache, f) in enumerate(((k, s["kc"], s["ks"]), (v, s["vc"], s["vs"]))):
        code, byte = _quantise(x, c["scaled"], f)
        _store(cache, s["sc"], i, c["page"], loc, code, byte)


def _turn(x, cs, rot, neox):
    """RoPE of rows x (f32) on their first rot dims."""
    half = rot // 2
    c, si = cs[:, None, :half], cs[:, None, half:rot]
    r = x[..., :rot]
    x0, x1 = (r[..., :half], r[..., half:]) if neox else (r[..., 0::2], r[..., 1::2])
    y0, y1 = x0 * c - x1 * si, x1 * c + x0 * si
    y = torch.cat([y0, y1], -1) if neox else torch.stack([y0, y1], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_rope(s):
    c = s["case"]
    cs = s["cs"][s["pos"].long()]
    _plain_write(s, _turn(s["k"].float(), cs, c["rot"], c["neox"]), s["v"])
    return _turn(s["q"].float(), cs, c["rot"], c["neox"]).to(s["q"].dtype)


def _plain_read(s):
    c = s["case"]
    loc, page, out = s["loc"].long(), c["page"], []
    for i, (cache, f) in enumerate(((s["kc"], s["ks"]), (s["vc"], s["vs"]))):
        x = _bits(cache)[loc // page, loc % page].view(F8).float()
        x = x * _power(s["sc"][loc // page, :, loc % page, i])[..., None] if s["sc"] is not None else x * f
        out.append(x.to(TYPES[c["dtype"]]))
    return out


def _cached(s, cache, i, f, page, slot):
    """Rows [B, Hkv, L, D] of a padded index [B, L], in f32."""
    x = _bits(cache)[page, slot].transpose(1, 2).contiguous().view(cache.dtype).float()
    if s["sc"] is not None:
        return x.mul_(_power(s["sc"][page, :, slot, i]).transpose(1, 2)[..., None])
    return x.mul_(f) if f != 1.0 else x


def _plain_attn(s):
    c = s["case"]
    q, qo, lens = s["q"], s["qo"].long(), s["lens"].long()
    b, hq, hkv, d, p = c["batch"], c["hq"], c["hkv"], c["d"], c["page"]
    g, (n, most) = hq // hkv, s["most"]
    key = torch.arange(most, device=DEV)
    row = torch.arange(n, device=DEV)
    new = qo[1:] - qo[:-1]
    real = row < new[:, None]
    pos = (lens - new)[:, None] + row
    page = s["table"].long()[:, key // p].clamp(min=0)
    slot = (key % p).expand(b, most)
    # [B, Hkv, rows * G, D]
    qp = q[(qo[:-1, None] + row).clamp(max=q.shape[0] - 1)].float().view(b, n, hkv, g, d).transpose(1, 2).reshape(b, hkv, n * g, d)
    w = torch.matmul(qp, _cached(s, s["kc"], 0, s["ks"], page, slot).transpose(2, 3)).view(b, hkv, n, g, most)
    w.mul_(s["sm"])
    if c["cap"]:
        w.div_(c["cap"]).tanh_().mul_(c["cap"])
    off = key > pos[..., None]
    if c["window"] >= 0:
        off |= key < pos[..., None] - c["window"]
    w.masked_fill_(off[:, None, :, None, :], -math.inf)
    m = w.amax(-1, keepdim=True).clamp(min=-3e38)
    w.sub_(m).exp_()
    total = w.sum(-1, keepdim=True)
    v = _cached(s, s["vc"], 1, s["vs"], page, slot)
    v.mul_((key < lens[:, None])[:, None, :, None])
    out = torch.matmul(w.view(b, hkv, n * g, most), v).view(b, hkv, n, g, d) / total
    lse = (m + total.log()).squeeze(-1)
    return out.transpose(1, 2)[real].reshape(-1, hq, d).to(q.dtype), lse.transpose(1, 2)[real].reshape(-1, hq)


# --------------------------------------------------------------------- run ---


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        ext = _ext()
        if op == "attn":
            return ext.mac_paged_chunk_attention(s["q"], s["kc"], s["vc"], s["qo"], s["lens"], s["table"], s["sm"],
                                                 kv_scales=s["sc"], k_scale=s["ks"], v_scale=s["vs"],
                                                 window_left=c["window"], logit_cap=c["cap"])
        if op == "read":
            return ext.mac_paged_cache_read_fp8(s["kc"], s["vc"], s["sc"], s["loc"], dtype=TYPES[c["dtype"]],
                                                k_scale=s["ks"], v_scale=s["vs"])
        if op == "write":
            ext.mac_paged_cache_write_fp8(s["k"], s["v"], s["kc"], s["vc"], s["sc"], s["loc"], k_scale=s["ks"],
                                          v_scale=s["vs"])
            return [s["kc"], s["vc"]] + ([s["sc"]] if c["scaled"] else [])
        q = ext.mac_paged_rope_write_fp8(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["sc"], s["cs"], s["pos"], s["loc"],
                                         is_neox=c["neox"], k_scale=s["ks"], v_scale=s["vs"])
    else:
        if op == "attn":
            return _plain_attn(s)
        if op == "read":
            return _plain_read(s)
        if op == "write":
            _plain_write(s, s["k"], s["v"])
            return [s["kc"], s["vc"]] + ([s["sc"]] if c["scaled"] else [])
        q = _plain_rope(s)
    return [s["kc"], s["vc"]] + ([s["sc"]] if c["scaled"] else []) + [q]


def work(case):
    if case["op"] == "attn":
        new, keys = _lengths(case)
        hq, hkv, d, w = case["hq"], case["hkv"], case["d"], case["window"]
        row = 2 * (d * (2 if case["cache"] == "same" else 1) + (1 if case["cache"] == "fp8" else 0))
        read = pairs = 0
        for n, k in zip(new, keys):
            first = k - n
            read += k if w < 0 else k - max(0, first - w)
            if w < 0:
                pairs += n * first + n * (n + 1) // 2
            else:
                full = max(0, min(n, k - w))  # rows whose whole window lies in the cache
                short = n - full
                pairs += full * (w + 1) + short * first + short * (short + 1) // 2
        # the rows in and out, the lse, the table
        moved = read * hkv * row + sum(new) * hq * (4 * d + 4) + 4 * sum(-(-k // case["page"]) for k in keys)
        return {"bytes": moved, "flops": 4 * d * hq * pairs}
    n, hkv, d = case["tokens"], case["hkv"], case["d"]
    cache = n * hkv * 2 * (d + (1 if case["scaled"] else 0)) + (8 if n % 2 else 4) * n
    elements = n * hkv * d * 2
    if case["op"] == "read":
        return {"bytes": cache + elements * (4 if case["dtype"] == "f32" else 2), "flops": elements}
    if case["op"] == "write":
        return {"bytes": cache + elements * 2, "flops": 4 * elements}
    q = n * case["hq"] * d
    return {"bytes": cache + elements * 2 + 4 * q + n * (4 * case["rot"] + (8 if n % 2 else 4)), "flops": 4 * elements + 3 * q}


# ------------------------------------------------------------------- exact ---


def _nearest(x):
    """The e4m3 value nearest to x (f64), ties to even, at most 448."""
    size = x.abs()
    step = torch.exp2(torch.floor(torch.log2(size.clamp(min=2.0 ** -6))) - 3)
    y = (torch.round(size / step) * step).clamp(max=448.0)
    return torch.where(x.isfinite(), torch.copysign(y, x), math.nan)


def _exact_rows(x, scaled, factor):
    x = x.double()
    if not scaled:
        return _nearest(x / factor), None
    size = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    e = torch.ceil(torch.log2((size / 448.0).clamp(min=2.0 ** -126))).long()
    e = torch.where(size > 448.0 * torch.exp2(e.double()), e + 1, e)
    e = torch.where((size <= 448.0 * torch.exp2(e.double() - 1)) & (e > -126), e - 1, e)
    return _nearest(x * torch.exp2(-e.double())[..., None]), e + 127


def _exact_values(cache, sc, i, f, flat):
    """Rows of flat slots in f64."""
    x = cache.view(-1, *cache.shape[2:])[flat].double() if cache.dtype != F8 else _bits(cache).view(
        -1, *cache.shape[2:])[flat].view(F8).double()
    if sc is None:
        return x * f
    byte = sc.transpose(1, 2).reshape(-1, sc.shape[1], 2)[flat][..., i]
    return x * torch.exp2(byte.double() - 127)[..., None]


def _exact_attn(case, s):
    d, hq, hkv, page = case["d"], case["hq"], case["hkv"], case["page"]
    g = hq // hkv
    new, keys = _lengths(case)
    out, lse, at = [], [], 0
    for i, (n, k) in enumerate(zip(new, keys)):
        key = torch.arange(k, device=DEV)
        flat = s["table"][i].long()[torch.div(key, page, rounding_mode="floor")] * page + key % page
        kk, vv = _exact_values(s["kc"], s["sc"], 0, s["ks"], flat), _exact_values(s["vc"], s["sc"], 1, s["vs"], flat)
        pos = torch.arange(k - n, k, device=DEV)[:, None]
        seen = key <= pos
        if case["window"] >= 0:
            seen &= key >= pos - case["window"]
        o, l = torch.empty(n, hq, d, device=DEV, dtype=torch.float64), torch.empty(n, hq, device=DEV, dtype=torch.float64)
        for h in range(hq):
            w = s["q"][at:at + n, h].double() @ kk[:, h // g].T.contiguous() * s["sm"]
            if case["cap"]:
                w = case["cap"] * torch.tanh(w / case["cap"])
            w = torch.where(seen, w, -math.inf)
            l[:, h] = torch.logsumexp(w, -1)
            o[:, h] = torch.exp(w - l[:, h, None]) @ vv[:, h // g].contiguous()
        out.append(o)
        lse.append(l)
        at += n
    return torch.cat(out), torch.cat(lse)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attn(case, s)
    page, loc = case["page"], s["loc"].long()
    if case["op"] == "read":
        return [_exact_values(s["kc"], s["sc"], 0, s["ks"], loc), _exact_values(s["vc"], s["sc"], 1, s["vs"], loc)]
    scaled, q = case["scaled"], None
    k, v = s["k"].double(), s["v"].double()
    if case["op"] == "rope":
        rot, half = case["rot"], case["rot"] // 2
        turn = torch.polar(torch.ones(1, device=DEV, dtype=torch.float64), torch.zeros(1, device=DEV, dtype=torch.float64))
        cs = s["cs"][s["pos"].long()].double()
        turn = turn * torch.complex(cs[:, :half], cs[:, half:])[:, None, :]
        done = []
        for x in (s["q"].double(), k):
            r = x[..., :rot]
            z = torch.complex(r[..., :half], r[..., half:]) if case["neox"] else torch.complex(r[..., 0::2], r[..., 1::2])
            z = z * turn
            y = torch.cat([z.real, z.imag], -1) if case["neox"] else torch.stack([z.real, z.imag], -1).flatten(-2)
            done.append(torch.cat([y, x[..., rot:]], -1))
        q, k = done
    outs = []
    sc = s["sc"].long() if scaled else None
    for i, (x, cache, f) in enumerate(((k, s["kc"], s["ks"]), (v, s["vc"], s["vs"]))):
        code, byte = _exact_rows(x, scaled, f)
        full = cache.double().view(-1, *cache.shape[2:])
        full[loc] = code
        outs.append(full.view(cache.shape))
        if scaled:
            sc[loc // page, :, loc % page, i] = byte
    return outs + ([sc] if scaled else []) + ([q] if q is not None else [])
