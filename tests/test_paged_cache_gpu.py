"""The 8-bit paged cache on the GPU: rows quantised as they are written, decode
RoPE with the write, rows read back -- against the format's definition in 64
bits.  Codes and scale bytes have to be equal; the one rounding of a code is
nearest-even, and every other step is exact (a static scale's quotient is an IEEE
fp32 division in both)."""

import math

import pytest
import torch

import paged_helpers as ph

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ext():
    from mac_attention.integrations.sglang.bridge import load_mac_paged_cache_extension

    return load_mac_paged_cache_extension(False)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _empty_cache(gen, pages, page, hkv, d, scaled):
    kc, vc = (torch.randint(0, 127, (pages, page, hkv, d), generator=gen, device=DEV, dtype=torch.uint8).view(ph.F8)
              for _ in range(2))
    sc = torch.randint(1, 255, (pages, hkv, page, 2), generator=gen, device=DEV, dtype=torch.uint8) if scaled else None
    return kc, vc, sc


def _rows(gen, n, h, d, dtype):
    return (torch.randn(n, h, d, generator=gen, device=DEV) * torch.exp2(3 * torch.randn(n, h, 1, generator=gen, device=DEV))).to(dtype)


def _expect_write(before, k, v, loc, page, scaled, ks=1.0, vs=1.0):
    kc, vc, sc = (None if t is None else t.clone() for t in before)
    ok = (loc >= 0) & (loc < kc.shape[0] * page)
    at = loc[ok].long()
    for i, (x, c, f) in enumerate(((k, kc, ks), (v, vc, vs))):
        code, byte = ph.quantise(x[ok], scaled, f)
        c.view(torch.uint8)[at // page, at % page] = code
        if scaled:
            sc[at // page, :, at % page, i] = byte
    return kc, vc, sc


def _same_codes(got, want, what):
    g, w = got.view(torch.uint8), want.view(torch.uint8)
    # (either NaN code is NaN)
    bad = (g != w) & ~((g & 127 == 127) & (w & 127 == 127))
    assert not bad.any(), f"{what}: {int(bad.sum())} codes differ, first at {bad.nonzero()[0].tolist()}"


def _check(got, want):
    _same_codes(got[0], want[0], "k_cache")
    _same_codes(got[1], want[1], "v_cache")
    if want[2] is not None:
        assert torch.equal(got[2], want[2]), "kv_scales differ"


@pytest.mark.parametrize("scaled", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hkv,d,page,loc64", [
    (1, 1, 16, 1, False), (1, 8, 128, 1, True), (7, 3, 64, 4, False), (64, 8, 128, 16, False), (333, 2, 256, 64, True),
    (50, 5, 80, 8, False), (129, 1, 240, 32, True), (17, 4, 48, 2, False)])
def test_write(ext, tokens, hkv, d, page, loc64, dtype, scaled):
    g = _gen(tokens * 31 + d)
    pages = -(-tokens // page) + 3
    cache = _empty_cache(g, pages, page, hkv, d, scaled)
    k, v = _rows(g, tokens, hkv, d, dtype), _rows(g, tokens, hkv, d, dtype)
    loc = torch.randperm(pages * page, generator=g, device=DEV)[:tokens].to(torch.int64 if loc64 else torch.int32)
    f = (1.0, 1.0) if scaled else (0.7, 0.031)
    want = _expect_write(cache, k, v, loc, page, scaled, *f)
    ext.mac_paged_cache_write_fp8(k, v, *cache, loc, k_scale=f[0], v_scale=f[1])
    _check(cache, want)


def test_write_every_16_bit_value(ext):
    """Each bf16 and fp16 value (NaN, infinities, subnormals among them), as rows
    of like exponents and as rows that mix them."""
    for dtype in (torch.bfloat16, torch.float16):
        bits = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16).view(dtype)
        mixed = bits[torch.randperm(65536, generator=_gen(3), device=DEV)]
        for x in (bits.view(-1, 1, 128), mixed.view(-1, 1, 128), mixed.view(-1, 4, 64)):
            n, h, d = x.shape
            cache = _empty_cache(_gen(1), n, 1, h, d, True)
            loc = torch.arange(n, device=DEV, dtype=torch.int32)
            want = _expect_write(cache, x, x.flip(0), loc, 1, True)
            ext.mac_paged_cache_write_fp8(x, x.flip(0), *cache, loc)
            _check(cache, want)
            cache = _empty_cache(_gen(2), n, 1, h, d, False)
            want = _expect_write(cache, x, x, loc, 1, False, 3.0, 1e-3)
            ext.mac_paged_cache_write_fp8(x, x, *cache, loc, k_scale=3.0, v_scale=1e-3)
            _check(cache, want)


def test_write_zero_rows_and_scale_borders(ext):
    """A row of zeros has the smallest scale; a row's largest element on, just
    under and just over 448 2^e."""
    x = torch.zeros(12, 1, 64, device=DEV, dtype=torch.bfloat16)
    for i, top in enumerate((448.0, 450.0, 446.0, 447.0, 1.75, 1.7578125, 1.7421875, 2.0 ** -120, 3e38, 896.0, 900.0)):
        x[i + 1, 0, 5] = top
        x[i + 1, 0, 9] = -top / 3
    cache = _empty_cache(_gen(0), 12, 1, 1, 64, True)
    loc = torch.arange(12, device=DEV, dtype=torch.int32)
    want = _expect_write(cache, x, -x, loc, 1, True)
    ext.mac_paged_cache_write_fp8(x, -x, *cache, loc)
    _check(cache, want)
    assert int(cache[2][0, 0, 0, 0]) == 1 and int(cache[2][1, 0, 0, 0]) == 127 and int(cache[2][2, 0, 0, 0]) == 128


def test_write_skips_locs_outside_and_leaves_the_rest(ext):
    g = _gen(9)
    cache = _empty_cache(g, 4, 8, 2, 64, True)
    k, v = _rows(g, 9, 2, 64, torch.bfloat16), _rows(g, 9, 2, 64, torch.bfloat16)
    loc = torch.tensor([-1, 3, 32, 31, 1 << 40, -(1 << 40), 0, -1, 17], device=DEV)
    want = _expect_write(cache, k, v, loc, 8, True)
    ext.mac_paged_cache_write_fp8(k, v, *cache, loc)
    _check(cache, want)


@pytest.mark.parametrize("layout", ["hnd", "interleaved", "wide"])
def test_write_and_read_other_layouts(ext, layout):
    """Pages of [Hkv, page, D], K and V interleaved, rows further apart; input
    rows that do not start on 16 bytes, heads in another order."""
    g = _gen(4)
    pages, page, hkv, d, n = 5, 8, 3, 64, 33
    kc, vc, sc = _empty_cache(g, pages, page, hkv, d, True)
    if layout == "hnd":
        kc, vc = (c.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(ph.F8) for c in (kc, vc))
    elif layout == "interleaved":
        both = torch.stack([kc.view(torch.uint8), vc.view(torch.uint8)], 1).contiguous()
        kc, vc = both[:, 0].view(ph.F8), both[:, 1].view(ph.F8)
    else:
        wide = torch.zeros(pages, page + 1, hkv + 1, d + 16, dtype=torch.uint8, device=DEV).view(ph.F8)
        kc, vc = wide[:, :page, :hkv, :d], wide.clone()[:, 1:, 1:, 16:]
    base = torch.randn(n, 2 * hkv, d + 3, generator=g, device=DEV).bfloat16()
    k, v = base[:, :hkv, 1:d + 1], base[:, hkv:, 3:].flip(1)
    loc = torch.randperm(pages * page, generator=g, device=DEV)[:n]
    want = _expect_write((kc, vc, sc), k, v, loc, page, True)
    ext.mac_paged_cache_write_fp8(k, v, kc, vc, sc, loc)
    _check((kc, vc, sc), want)
    out = ext.mac_paged_cache_read_fp8(kc, vc, sc, loc, dtype=torch.float32)
    for x, y in zip((k, v), out):
        code, byte = ph.quantise(x, True)
        assert torch.equal(y.double(), ph.values(code, byte, 1.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scaled", [True, False])
@pytest.mark.parametrize("rows,hkv,d,page", [(1, 1, 16, 1), (5, 8, 128, 16), (200, 2, 256, 64), (77, 3, 112, 2), (64, 4, 64, 8)])
def test_read(ext, rows, hkv, d, page, scaled, dtype):
    g = _gen(rows + d)
    pages = 7 + rows // page
    kc, vc, sc = _empty_cache(g, pages, page, hkv, d, scaled)
    if scaled:  # rows in the outputs' range, and NaN and tiny scales
        sc.copy_(torch.randint(120, 130, sc.shape, generator=g, device=DEV, dtype=torch.uint8))
        sc[0], sc[1] = 255, 1
    kc.view(torch.uint8)[2, 0, 0, :4] = torch.tensor([127, 255, 0, 128], dtype=torch.uint8, device=DEV)
    idx = torch.randint(-3, pages * page + 3, (rows,), generator=g, device=DEV).to(torch.int32 if rows % 2 else torch.int64)
    f = (1.0, 1.0) if scaled else (0.3, 7.0)
    got = ext.mac_paged_cache_read_fp8(kc, vc, sc, idx, dtype=dtype, k_scale=f[0], v_scale=f[1])
    ok = (idx >= 0) & (idx < pages * page)
    at = torch.where(ok, idx, 0).long()
    for i, (c, out) in enumerate(zip((kc, vc), got)):
        byte = sc[at // page, :, at % page, i] if scaled else None
        want = ph.values(c.view(torch.uint8)[at // page, at % page], byte, float(torch.tensor(f[i])))
        if byte is not None:
            want = torch.where((byte == 255)[..., None], math.nan, want)
        want = torch.where(ok[:, None, None], want, 0.0)
        # (exact in fp32 when scaled; a static product rounds to fp32, then to dtype)
        want = want.float().to(dtype)
        assert torch.equal(out.nan_to_num(12345.0), want.nan_to_num(12345.0))
        assert torch.equal(out.isnan(), want.isnan())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hq,hkv,d,rot,page,neox,scaled", [
    (1, 4, 1, 128, 128, 1, True, True), (64, 32, 8, 128, 128, 16, True, True), (9, 6, 2, 64, 32, 4, False, False),
    (33, 5, 5, 256, 256, 8, True, True), (20, 4, 2, 96, 20, 2, True, True), (20, 4, 2, 96, 22, 2, False, True),
    (16, 7, 1, 80, 64, 1, False, True), (5, 2, 2, 128, 48, 1, True, False)])
def test_rope_write(ext, tokens, hq, hkv, d, rot, page, neox, scaled, dtype):
    g = _gen(tokens + rot)
    pages = -(-tokens // page) + 2
    cache = _empty_cache(g, pages, page, hkv, d, scaled)
    qkv = _rows(g, tokens, hq + 2 * hkv, d, dtype)
    q, k, v = qkv.split([hq, hkv, hkv], dim=1)
    keep = qkv.clone()
    cs = torch.randn(500, rot, generator=g, device=DEV)
    pos = torch.randint(-2, 502, (tokens,), generator=g, device=DEV)
    loc = torch.randperm(pages * page, generator=g, device=DEV)[:tokens].to(torch.int32)
    f = (1.0, 1.0) if scaled else (0.4, 0.9)
    row = cs[pos.clamp(0, 499)]

    def turn(x):
        # fp32 products and sums, each rounded on its own: the keys' codes
        # follow from these bits
        x, half = x.float().clone(), rot // 2
        c, s = row[:, None, :half], row[:, None, half:]
        r = x[..., :rot].clone()
        x0, x1 = (r[..., :half], r[..., half:]) if neox else (r[..., 0::2], r[..., 1::2])
        y0, y1 = x0 * c - x1 * s, x1 * c + x0 * s
        x[..., :rot] = torch.cat([y0, y1], -1) if neox else torch.stack([y0, y1], -1).flatten(-2)
        return x

    want = _expect_write(cache, turn(k), v.float(), loc, page, scaled, *f)
    got = ext.mac_paged_rope_write_fp8(q, k, v, *cache, cs, pos, loc, is_neox=neox, k_scale=f[0], v_scale=f[1])
    assert torch.equal(got, turn(q).to(dtype))
    assert torch.equal(qkv, keep)  # the inputs stay: q is the pre-RoPE query
    _check(cache, want)


def test_rope_write_misaligned_inputs_and_tables(ext):
    g = _gen(11)
    n, d = 12, 64
    base = torch.randn(n, 4, d + 1, generator=g, device=DEV).bfloat16()
    q, k, v = base[:, :2, 1:], base[:, 2:3, 1:], base[:, 3:, :d]
    cs = torch.randn(40, d + 1, generator=g, device=DEV)[:, 1:]
    pos = torch.arange(n, device=DEV, dtype=torch.int32)
    loc = torch.arange(n, device=DEV)
    cache = _empty_cache(g, 3, 4, 1, d, True)
    plain = [t.clone() for t in cache]
    a = ext.mac_paged_rope_write_fp8(q, k, v, *cache, cs, pos, loc)
    b = ext.mac_paged_rope_write_fp8(q.contiguous(), k.contiguous(), v.contiguous(), *plain, cs.contiguous(), pos, loc)
    assert torch.equal(a, b)
    _check(cache, plain)


def test_empty_calls(ext):
    cache = _empty_cache(_gen(1), 2, 4, 2, 64, True)
    none = torch.empty(0, 2, 64, device=DEV, dtype=torch.bfloat16)
    idx = torch.empty(0, device=DEV, dtype=torch.int32)
    ext.mac_paged_cache_write_fp8(none, none, *cache, idx)
    k, v = ext.mac_paged_cache_read_fp8(*cache, idx)
    assert k.shape == (0, 2, 64) and v.shape == (0, 2, 64)
    q = ext.mac_paged_rope_write_fp8(none, none, none, *cache, torch.zeros(3, 64, device=DEV), idx, idx)
    assert q.shape == (0, 2, 64)


def test_slots_past_32_bit_offsets(ext):
    """A cache of more than 2^32 bytes: rows at its end."""
    page, hkv, d = 16, 8, 128
    pages = (1 << 32) // (page * hkv * d) + 8
    kc, vc = (torch.zeros(pages, page, hkv, d, dtype=torch.uint8, device=DEV).view(ph.F8) for _ in range(2))
    sc = torch.full((pages, hkv, page, 2), 127, dtype=torch.uint8, device=DEV)
    g = _gen(5)
    k, v = _rows(g, 40, hkv, d, torch.bfloat16), _rows(g, 40, hkv, d, torch.bfloat16)
    loc = pages * page - 1 - torch.arange(40, device=DEV)
    ext.mac_paged_cache_write_fp8(k, v, kc, vc, sc, loc)
    out = ext.mac_paged_cache_read_fp8(kc, vc, sc, loc, dtype=torch.float32)
    for x, y in zip((k, v), out):
        code, byte = ph.quantise(x, True)
        assert torch.equal(y.double(), ph.values(code, byte, 1.0))
    assert not kc.view(torch.uint8)[:64].any()


def test_captured_and_on_another_stream(ext):
    """A decode step's write in a graph, replayed over changing inputs with eager
    work between the replays; a call on a side stream."""
    g = _gen(6)
    n, hq, hkv, d, page = 16, 8, 2, 128, 4
    cache = _empty_cache(g, 8, page, hkv, d, True)
    q, k, v = _rows(g, n, hq, d, torch.bfloat16), _rows(g, n, hkv, d, torch.bfloat16), _rows(g, n, hkv, d, torch.bfloat16)
    cs = torch.randn(64, d, generator=g, device=DEV)
    pos = torch.randint(0, 64, (n,), generator=g, device=DEV)
    loc = torch.randperm(32, generator=g, device=DEV)[:n]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ext.mac_paged_rope_write_fp8(q, k, v, *cache, cs, pos, loc)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ext.mac_paged_rope_write_fp8(q, k, v, *cache, cs, pos, loc)
        rk, rv = ext.mac_paged_cache_read_fp8(*cache, loc)
    for i in range(4):
        k.copy_(_rows(g, n, hkv, d, torch.bfloat16))
        q.copy_(_rows(g, n, hq, d, torch.bfloat16))
        loc.copy_(torch.randperm(32, generator=g, device=DEV)[:n])
        plain = [t.clone() for t in cache]
        want = ext.mac_paged_rope_write_fp8(q, k, v, *plain, cs, pos, loc)
        wk, wv = ext.mac_paged_cache_read_fp8(*plain, loc)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(rk, wk) and torch.equal(rv, wv)
        _check(cache, plain)


def test_refusals(ext):
    g = _gen(0)
    cache = _empty_cache(g, 4, 8, 2, 64, True)
    kc, vc, sc = cache
    k = _rows(g, 3, 2, 64, torch.bfloat16)
    loc = torch.arange(3, device=DEV)
    w = ext.mac_paged_cache_write_fp8

    def refused(text, fn, *args, **kw):
        with pytest.raises(RuntimeError, match=text):
            fn(*args, **kw)

    refused("must be CUDA", w, k.cpu(), k, kc, vc, sc, loc)
    refused("bfloat16 or float16", w, k.float(), k.float(), kc, vc, sc, loc)
    refused("must match k", w, k, k[:2], kc, vc, sc, loc)
    refused("must match k", w, k, k.half(), kc, vc, sc, loc)
    refused("wrong shape", w, k[..., :32], k[..., :32], kc, vc, sc, loc)
    refused("contiguous last", w, k.transpose(1, 2).contiguous().transpose(1, 2), k, kc, vc, sc, loc)
    refused("wrong length", w, k, k, kc, vc, sc, loc[:2])
    refused("wrong dtype", w, k, k, kc, vc, sc, loc.float())
    refused("float8_e4m3fn", w, k, k, kc.view(torch.float8_e5m2), vc, sc, loc)
    refused("v_cache must have", w, k, k, kc, vc.view(torch.uint8), sc, loc)
    refused("uint8", w, k, k, kc, vc, sc.int(), loc)
    refused("contiguous \\[pages", w, k, k, kc, vc, sc[:3], loc)
    refused("k_scale", w, k, k, kc, vc, sc, loc, k_scale=2.0)
    refused("positive", w, k, k, kc, vc, None, loc, k_scale=0.0)
    refused("positive", w, k, k, kc, vc, None, loc, v_scale=float("nan"))
    refused("power of two", w, k, k, kc[:, :6], vc[:, :6], torch.zeros(4, 2, 6, 2, dtype=torch.uint8, device=DEV), loc)
    refused("multiple of 16", w, k[..., :40], k[..., :40], kc[..., :40], vc[..., :40], sc, loc)
    odd = torch.zeros(4 * 8 * 2 * 64 + 16, dtype=torch.uint8, device=DEV)[8:-8].view(ph.F8).view(4, 8, 2, 64)
    refused("16-byte aligned", w, k, k, odd, vc, sc, loc)
    wide = torch.zeros(4, 8, 2, 72, dtype=torch.uint8, device=DEV).view(ph.F8)[..., :64]
    refused("multiples of 16", w, k, k, wide, vc, sc, loc)
    r = ext.mac_paged_cache_read_fp8
    refused("dtype must be", r, kc, vc, sc, loc, dtype=torch.float64)
    refused("out_k", r, kc, vc, sc, loc, out_k=torch.empty(2, 2, 64, device=DEV, dtype=torch.bfloat16))
    rope = ext.mac_paged_rope_write_fp8
    cs = torch.zeros(8, 64, device=DEV)
    refused("invalid rotary_dim", rope, k, k, k, kc, vc, sc, cs[:, :7], loc, loc)
    refused("same dtype", rope, k.half(), k, k, kc, vc, sc, cs, loc, loc)
    refused("batch mismatch", rope, k[:2], k, k, kc, vc, sc, cs, loc, loc)
    refused("wrong length", rope, k, k, k, kc, vc, sc, cs, loc[:1], loc)
    refused("not be empty", rope, k, k, k, kc, vc, sc, cs[:0], loc, loc)
    # a scale tensor of the E8M0 type is taken
    w(k, k, kc, vc, sc.view(torch.float8_e8m0fnu), loc)
