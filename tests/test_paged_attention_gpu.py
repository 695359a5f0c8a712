"""Attention of a chunk of new tokens over a paged cache, on the GPU, against
softmax attention in 64 bits (tolerances: paged_helpers.attention)."""

import math

import pytest
import torch

import paged_helpers as ph

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, H = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ext():
    from mac_attention.integrations.sglang.bridge import load_mac_paged_cache_extension

    return load_mac_paged_cache_extension(False)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(xs):
    return torch.tensor(xs, device=DEV, dtype=torch.int32)


class Problem:
    """Requests of `new` rows over `lens` keys, and their oracle."""

    def __init__(self, new, lens, hq, hkv, d, page, kind="fp8", dtype=BF, window=-1, cap=0.0, seed=0, layout="nhd", qscale=1.0):
        g = _gen(seed)
        self.new, self.lens, self.page, self.window, self.cap = new, lens, page, window, cap
        self.table, pages = ph.page_table(g, lens, page, DEV)
        self.kc, self.vc, self.sc, self.ks, self.vs, self.k, self.v = ph.make_cache(g, pages, page, hkv, d, kind, dtype, DEV, layout)
        self.q = (qscale * torch.randn(sum(new), hq, d, generator=g, device=DEV)).to(dtype)
        self.qo, self.kv_lens = _i32(ph.offsets(new)), _i32(lens)
        self.sm = 1 / math.sqrt(d)
        self.req_ids = None

    def run(self, ext, **kw):
        args = dict(kv_scales=self.sc, k_scale=self.ks, v_scale=self.vs, window_left=self.window, logit_cap=self.cap,
                    req_ids=None if self.req_ids is None else _i32(self.req_ids))
        args.update(kw)
        return ext.mac_paged_chunk_attention(self.q, self.kc, self.vc, self.qo, self.kv_lens, self.table, self.sm, **args)

    def want(self):
        return ph.attention(self.q, self.k, self.v, self.new, self.lens, self.table, self.page, self.kc.shape[0], self.sm,
                            self.window, self.cap, self.req_ids)

    def check(self, got):
        out, lse, to, tl = self.want()
        ph.assert_close(got[0], out, to, "out")
        ph.assert_close(got[1], lse, tl, "lse")


KINDS = [("fp8", BF), ("fp8", H), ("static", BF), ("same", BF), ("same", H)]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("new,lens,hq,hkv,d,page", [
    ([1], [1], 1, 1, 64, 1),
    ([1], [333], 8, 2, 128, 1),
    ([1, 1, 1], [1, 4000, 129], 16, 2, 128, 16),
    ([1] * 9, [5, 64, 31, 32, 33, 128, 1000, 1, 257], 6, 2, 64, 4),
    ([1, 1], [700, 40], 16, 1, 256, 64),
    ([1, 1], [2500, 40], 40, 1, 128, 8),
    ([5, 5, 5], [64, 900, 5], 8, 1, 128, 16),
    ([3, 7], [300, 1500], 3, 1, 128, 2),
    ([4, 2, 9], [100, 2, 600], 14, 2, 64, 32),
    ([8, 8], [333, 1024], 8, 4, 256, 16),
    ([64], [64], 4, 2, 128, 16),
    ([100, 1, 37], [100, 500, 900], 8, 2, 128, 1),
    ([129, 64], [129, 700], 5, 1, 64, 8),
    ([200, 30], [1111, 30], 2, 2, 256, 32),
    ([300], [1500], 12, 4, 128, 256),
    ([70], [70], 200, 1, 128, 16),
])
def test_against_softmax(ext, new, lens, hq, hkv, d, page, kind, dtype):
    p = Problem(new, lens, hq, hkv, d, page, kind, dtype, seed=len(new) + d)
    p.check(p.run(ext))


@pytest.mark.parametrize("new", [[1, 1, 1], [6, 3, 11], [40, 90, 17]])
@pytest.mark.parametrize("window", [0, 1, 17, 63, 200])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("kind,d", [("fp8", 128), ("same", 64), ("static", 256)])
def test_windows_and_caps(ext, new, window, cap, kind, d):
    p = Problem(new, [700, 95, 333], 8, 2, d, 16, kind, window=window, cap=cap, seed=window, qscale=3.0)
    p.check(p.run(ext))


@pytest.mark.parametrize("d,kind,dtype", [(64, "fp8", BF), (128, "same", H), (256, "fp8", H), (128, "fp8", BF)])
@pytest.mark.parametrize("rows", [1, 12, 60])
def test_long_contexts_shared_by_many_workgroups(ext, rows, d, kind, dtype):
    p = Problem([rows, 1, rows], [9000, 20000, 70], 8, 2, d, 16, kind, dtype, seed=d)
    p.check(p.run(ext))


@pytest.mark.parametrize("rows", [2100, 4096])
def test_whole_prompts(ext, rows):
    p = Problem([rows, 1300], [rows, 1300], 8, 8, 64, 16, "fp8", seed=rows)
    p.check(p.run(ext))


@pytest.mark.parametrize("window", [-1, 300])
@pytest.mark.parametrize("lens", [[1600, 40000, 900], [1600, 1, 0], [1700, 9000, 1601], [50000, 700, 3]])
def test_chunks_beside_single_tokens(ext, lens, window):
    """More tasks than resident workgroups, of lengths that only the device knows: of
    whole tasks, or streamed where one is much longer."""
    p = Problem([1600, 1, 1], lens, 64, 8, 64, 16, "fp8", window=window, seed=lens[1])
    p.check(p.run(ext))


def test_captured_while_the_longest_task_changes(ext):
    """Replays of one capture switch between whole and streamed tasks."""
    cases = [[1600, 40000], [1600, 900], [1600, 30000], [1600, 1]]
    p = Problem([1600, 1], cases[0], 64, 8, 64, 16, "fp8", seed=3)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        p.run(ext)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = p.run(ext)
    for lens in cases + cases:
        p.lens = lens
        p.kv_lens.copy_(_i32(lens))
        eager = [x.clone() for x in p.run(ext)]
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, eager):
            assert torch.equal(x, y)
    p.lens = cases[2]
    p.kv_lens.copy_(_i32(p.lens))
    graph.replay()
    p.check(got)


def test_many_requests(ext):
    """More requests than a workgroup has threads, some without rows."""
    g = torch.Generator().manual_seed(1)
    new = torch.randint(0, 3, (700,), generator=g).tolist()
    lens = [max(n, int(x)) for n, x in zip(new, torch.randint(1, 300, (700,), generator=g))]
    p = Problem(new, lens, 4, 2, 64, 8, seed=3)
    p.check(p.run(ext))


@pytest.mark.parametrize("rows", [1, 6, 50, 200])
def test_rows_without_keys(ext, rows):
    """Requests with no cached key, or fewer keys than new rows: those rows are 0
    and -inf, whatever the output held."""
    p = Problem([rows, rows, rows, rows], [0, rows // 2, rows, -3], 4, 2, 128, 16)
    out = torch.full_like(p.q, math.nan)
    lse = torch.full((p.q.shape[0], 4), math.nan, device=DEV)
    p.run(ext, out=out, out_lse=lse)
    p.check((out, lse))
    assert torch.all(out[:rows] == 0) and torch.all(lse[:rows] == -math.inf)


@pytest.mark.parametrize("rows", [1, 7, 150])
def test_pages_outside_the_pool_are_masked(ext, rows):
    p = Problem([rows, rows], [900, 500], 8, 2, 128, 16)
    p.table[0, 3] = -1
    p.table[0, 20] = p.kc.shape[0]
    p.table[1, 0] = 1 << 30
    p.table[1, 31] = -(1 << 31)  # the new rows' own page, in part
    p.check(p.run(ext))


@pytest.mark.parametrize("kind", ["fp8", "same"])
@pytest.mark.parametrize("rows,window", [(1, -1), (5, -1), (30, 40), (100, -1), (200, 90)])
def test_unused_slots_may_hold_anything(ext, kind, rows, window):
    """NaN and infinities in slots past a request's keys, in pages of nobody and
    in keys before every row's window."""
    p = Problem([rows, rows], [rows + 133, rows + 250], 8, 2, 128, 16, kind, window=window)
    want = p.run(ext)
    used = torch.zeros(p.kc.shape[0] * 16, dtype=torch.bool, device=DEV)
    for b, n in enumerate(p.lens):
        lo = 0 if window < 0 else max(n - rows - window, 0)
        key = torch.arange(lo, n, device=DEV)
        used[p.table[b].long()[key // 16] * 16 + key % 16] = True
    used = used.view(-1, 16)
    poison = 127 if kind == "fp8" else math.nan
    for c in (p.kc, p.vc):
        c = c.view(torch.uint8) if kind == "fp8" else c
        c[~used] = poison
        if kind == "same":
            c[3:][~used[3:]] = math.inf
    if p.sc is not None:
        p.sc.transpose(1, 2)[~used] = 255
    got = p.run(ext)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", ["fp8", "same"])
@pytest.mark.parametrize("rows", [4, 20, 64, 150])
@pytest.mark.parametrize("d", [64, 256])
def test_a_poisoned_token_spares_the_rows_before_it(ext, kind, rows, d):
    """A new token whose K and V are not finite reaches its own and later rows
    only (a masked weight of 0 times NaN would reach all)."""
    p = Problem([rows, rows], [rows + 77, rows], 4, 2, d, 16, kind)
    clean = p.run(ext)
    at = rows // 2
    for b, n in enumerate(p.lens):
        key = n - rows + at
        page, slot = int(p.table[b, key // 16]), key % 16
        for c, val in ((p.kc, math.nan), (p.vc, -math.inf)):
            if kind == "fp8":
                c.view(torch.uint8)[page, slot, :, 3] = 127
            else:
                c[page, slot, :, 3] = val
    out, lse = p.run(ext)
    mine = torch.cat([torch.arange(rows) < at] * 2).to(DEV)
    assert torch.equal(lse[mine], clean[1][mine])
    # (the poisoned block's product is summed apart for the rows before: fp32
    # weights, so it may differ by the weights' rounding)
    want = p.want()
    ph.assert_close(out[mine], want[0][mine], want[2][mine], "rows before")
    assert torch.isnan(out[~mine]).any(-1).all() and torch.isnan(lse[~mine]).all()


@pytest.mark.parametrize("rows", [4, 150])
def test_poisoned_values_alone(ext, rows):
    """V infinite at one new token (K finite): the rows that see it have that
    infinity in that dim, the others are untouched.  (The lse of the rows that see
    it sums the same terms in another order: l's fp32 sum of positive terms is
    within paged_helpers.attention's bound in any order, so it is held to that
    bound instead of the bits of a clean run.)"""
    p = Problem([rows], [rows + 40], 4, 2, 128, 16, "same")
    clean = p.run(ext)
    at, key = rows // 2, 40 + rows // 2
    p.vc[int(p.table[0, key // 16]), key % 16, :, 7] = math.inf
    out, lse = p.run(ext)
    assert torch.equal(lse[:at], clean[1][:at])
    assert torch.all(out[at:, :, 7] == math.inf)
    want = p.want()
    ph.assert_close(lse, want[1], want[3], "lse")
    ph.assert_close(out[:at], want[0][:at], want[2][:at], "rows before")
    keep = torch.arange(128, device=DEV) != 7
    p.vc[int(p.table[0, key // 16]), key % 16, :, 7] = 0
    want = p.want()
    ph.assert_close(out[at:][..., keep], want[0][at:][..., keep], want[2][at:][..., keep], "other dims")


@pytest.mark.parametrize("rows", [1, 9, 120])
def test_large_scores(ext, rows):
    """Rows whose scores lie far below or above 0, one of them past the running
    reference point's lazy bound many times over."""
    p = Problem([rows], [900], 4, 2, 128, 16, "same", qscale=30.0, seed=5)
    p.check(p.run(ext))
    p.k.neg_()
    p.kc.neg_()
    p.check(p.run(ext))


@pytest.mark.parametrize("rows", [1, 5, 70])
def test_lowest_values(ext, rows):
    """Every score near -3e38 (keys of the type's lowest values): still a
    softmax over them."""
    p = Problem([rows], [100], 2, 2, 64, 16, "same", seed=2)
    p.q.fill_(1.0)
    p.kc.fill_(torch.finfo(BF).min / 128)
    p.k.fill_(float(torch.tensor(torch.finfo(BF).min / 128).bfloat16()))
    out, lse = p.run(ext)
    want = p.want()
    # equal scores: the mean of the seen values
    ph.assert_close(out, want[0], want[2], "out")
    assert torch.all((lse.double() - want[1]).abs() <= 2.0 ** -20 * want[1].abs())


def test_req_ids_strided_queries_and_tables(ext):
    g = _gen(7)
    p = Problem([1, 5, 2], [200, 90, 700], 8, 2, 128, 16, seed=7)
    wide = torch.full((9, p.table.shape[1] + 5), -7, dtype=torch.int32, device=DEV)
    p.req_ids = [4, 8, 1]
    for b, r in enumerate(p.req_ids):
        wide[r, :p.table.shape[1]] = p.table[b]
    p.table = wide[:, :-2]
    p.check(p.run(ext))
    # queries as a slice of the fused projection, and as heads in another order
    qkv = torch.randn(8, 12, 128, generator=g, device=DEV).bfloat16()
    p.q = qkv[:, 2:10]
    p.check(p.run(ext))
    p.q = torch.randn(8, 8, 128, generator=g, device=DEV).bfloat16().transpose(0, 1)
    p.check(p.run(ext))
    p.q = torch.randn(8, 8, 129, generator=g, device=DEV).bfloat16()[..., 1:]  # rows not on 16 bytes
    p.check(p.run(ext))
    # a table row outside the table: no keys
    p.req_ids = [4, 9, -1]
    out, lse = p.run(ext)
    assert torch.all(out[1:] == 0) and torch.all(lse[1:] == -math.inf)


@pytest.mark.parametrize("layout", ["hnd", "interleaved"])
@pytest.mark.parametrize("kind,rows", [("fp8", 1), ("fp8", 70), ("same", 3), ("same", 200)])
def test_layouts(ext, layout, kind, rows):
    p = Problem([rows, rows], [rows + 300, rows + 17], 8, 2, 128, 32, kind, layout=layout)
    p.check(p.run(ext))


def test_kv_lens_past_the_table(ext):
    """More keys than the table can name: those past it are masked, positions
    stay the caller's."""
    p = Problem([2, 40], [500, 300], 4, 2, 64, 16)
    p.table = p.table[:, :10].contiguous()
    p.check(p.run(ext))


@pytest.mark.parametrize("rows", [1, 3, 64, 300])
def test_rows_of_no_request_are_left(ext, rows):
    """Rows before the first offset and behind the last, as in a padded batch."""
    p = Problem([rows, rows], [rows + 50, rows + 9], 4, 2, 128, 16)
    want = p.run(ext)
    pad = 5
    q = torch.cat([p.q[:pad % rows + 1], p.q, p.q[:1].expand(pad, -1, -1)])
    first = pad % rows + 1
    out, lse = torch.full_like(q, 7.0), torch.full((q.shape[0], 4), 7.0, device=DEV)
    ext.mac_paged_chunk_attention(q, p.kc, p.vc, p.qo + first, p.kv_lens, p.table, p.sm, kv_scales=p.sc, out=out, out_lse=lse)
    n = 2 * rows
    assert torch.all(out[:first] == 7) and torch.all(out[first + n:] == 7)
    assert torch.all(lse[:first] == 7) and torch.all(lse[first + n:] == 7)
    ref = p.want()
    ph.assert_close(out[first:first + n], ref[0], ref[2], "out")
    ph.assert_close(lse[first:first + n], ref[1], ref[3], "lse")
    del want


def test_bad_offsets_touch_nothing(ext):
    """Requests whose rows do not lie within q are skipped."""
    p = Problem([3, 3, 3], [50, 60, 70], 4, 2, 64, 16)
    for qo in ([0, 3, 100, 9], [-4, 3, 6, 9], [0, 3, 2, 9], [5, 5, 5, 5]):
        out, lse = torch.full_like(p.q, 7.0), torch.full((9, 4), 7.0, device=DEV)
        ext.mac_paged_chunk_attention(p.q, p.kc, p.vc, _i32(qo), p.kv_lens, p.table, p.sm, kv_scales=p.sc, out=out, out_lse=lse)
        torch.cuda.synchronize()
    assert torch.all(out == 7) and torch.all(lse == 7)


def test_cache_past_32_bit_offsets(ext):
    """Pages past 4 GiB of K."""
    page, hkv, d = 16, 8, 128
    pages = (1 << 32) // (page * hkv * d) + 40
    kc, vc = (torch.zeros(pages, page, hkv, d, dtype=torch.uint8, device=DEV).view(ph.F8) for _ in range(2))
    sc = torch.full((pages, hkv, page, 2), 127, dtype=torch.uint8, device=DEV)
    p = Problem([1, 4, 80], [300, 77, 100], 16, hkv, d, page)
    own = p.kc.shape[0]
    kc.view(torch.uint8)[-own:] = p.kc.view(torch.uint8)
    vc.view(torch.uint8)[-own:] = p.vc.view(torch.uint8)
    sc[-own:] = p.sc
    table = torch.where(p.table >= 0, p.table + (pages - own), p.table)
    out = ext.mac_paged_chunk_attention(p.q, kc, vc, p.qo, p.kv_lens, table, p.sm, kv_scales=sc)
    p.check(out)


def test_repeats_are_bitwise_equal(ext):
    for new, lens in (([1, 1], [9000, 300]), ([5, 5], [4000, 777]), ([300, 1], [2000, 90])):
        p = Problem(new, lens, 8, 2, 128, 16)
        a = p.run(ext)
        for _ in range(3):
            b = p.run(ext)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_with_lengths_that_grow(ext):
    """One graph of two layers' calls replayed while the contexts grow and the
    caches change, eager calls and synchronisations in between."""
    p = Problem([1, 1, 1], [900, 333, 64], 8, 2, 128, 16)
    p.check(p.run(ext))
    p.kv_lens.copy_(_i32([500, 100, 10]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = p.run(ext)
        b = p.run(ext, window_left=64)
    for step in range(5):
        lens = [500 + 97 * step, 100 + 50 * step, 10 + 13 * step]
        p.kv_lens.copy_(_i32(lens))
        p.lens = lens
        p.q.normal_()
        graph.replay()
        wa, wb = p.run(ext), p.run(ext, window_left=64)
        torch.cuda.synchronize()
        assert torch.equal(a[0], wa[0]) and torch.equal(a[1], wa[1])
        assert torch.equal(b[0], wb[0]) and torch.equal(b[1], wb[1])
        p.check(a)


def test_calls_on_two_streams(ext):
    ps = [Problem([1, 1], [6000, 100 + i], 8, 2, 128, 16, seed=i) for i in range(2)]
    want = [p.run(ext) for p in ps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    for _ in range(5):
        got = []
        for p, s in zip(ps, streams):
            with torch.cuda.stream(s):
                got.append(p.run(ext))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_serving_sequence(ext):
    """The operators as serving uses them: a prompt in two chunks written and
    attended to, decode steps with RoPE and the write, drafted tokens, and the
    prefix read back for a 16-bit kernel -- each against 64-bit attention over
    the values that the cache holds."""
    g = _gen(12)
    hq, hkv, d, page, b = 8, 2, 128, 16, 2
    pages = 24
    kc, vc = (torch.zeros(pages, page, hkv, d, dtype=torch.uint8, device=DEV).view(ph.F8) for _ in range(2))
    sc = torch.full((pages, hkv, page, 2), 127, dtype=torch.uint8, device=DEV)
    table = torch.randperm(pages, generator=g, device=DEV).int().view(b, -1)
    flat = (table.long()[:, :, None] * page + torch.arange(page, device=DEV)).flatten(1)
    pos_t = torch.arange(4096, device=DEV, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(0, d, 2, device=DEV) / d))
    cs = torch.cat([pos_t.cos(), pos_t.sin()], 1).float()
    lens = [0, 0]
    sm = d ** -0.5

    def step(new):
        n = sum(new)
        qkv = torch.randn(n, hq + 2 * hkv, d, generator=g, device=DEV).bfloat16()
        q, k, v = qkv.split([hq, hkv, hkv], dim=1)
        pos = torch.cat([torch.arange(l, l + m, device=DEV) for l, m in zip(lens, new)])
        loc = torch.cat([flat[i, l:l + m] for i, (l, m) in enumerate(zip(lens, new))])
        qr = ext.mac_paged_rope_write_fp8(q, k, v, kc, vc, sc, cs, pos, loc)
        for i, m in enumerate(new):
            lens[i] += m
        out = ext.mac_paged_chunk_attention(qr, kc, vc, _i32(ph.offsets(new)), _i32(lens), table, sm, kv_scales=sc)
        rows = [ph.values(c.view(torch.uint8).view(-1, hkv, d), sc.transpose(1, 2).reshape(-1, hkv, 2)[..., i], 1.0)
                for i, c in enumerate((kc, vc))]
        want = ph.attention(qr, *rows, new, lens, table, page, pages, sm)
        ph.assert_close(out[0], want[0], want[2], "out")
        ph.assert_close(out[1], want[1], want[3], "lse")

    for new in ([70, 20], [50, 1], [1, 1], [1, 1], [5, 5], [1, 1]):
        step(new)
    k16, v16 = ext.mac_paged_cache_read_fp8(kc, vc, sc, flat[0, :lens[0]].contiguous())
    k32, _ = ext.mac_paged_cache_read_fp8(kc, vc, sc, flat[0, :lens[0]].contiguous(), dtype=torch.float32)
    assert torch.equal(k16.float(), k32)  # exact in bf16
    # the same attention over the rows read back, as a 16-bit cache
    q = torch.randn(1, hq, d, generator=g, device=DEV).bfloat16()
    ident = torch.arange(lens[0], device=DEV, dtype=torch.int32)[None]
    a = ext.mac_paged_chunk_attention(q, kc, vc, _i32([0, 1]), _i32(lens[:1]), table[:1], sm, kv_scales=sc)
    c = ext.mac_paged_chunk_attention(q, k16.unsqueeze(1), v16.unsqueeze(1), _i32([0, 1]), _i32(lens[:1]), ident, sm)
    want = ph.attention(q, k16.double(), v16.double(), [1], lens[:1], ident, 1, lens[0], sm)
    for got in (a, c):
        ph.assert_close(got[0], want[0], want[2], "out")
        ph.assert_close(got[1], want[1], want[3], "lse")


def test_against_the_window_kernel(ext):
    """The framework's bf16 window attention over the same pool."""
    from mac_attention.integrations.sglang.bridge import load_mac_prefill_rectify_extension

    rect = load_mac_prefill_rectify_extension(False)
    p = Problem([40, 3], [300, 90], 8, 2, 128, 1, "same", window=99)
    kv_indices = torch.cat([p.table[b, :n] for b, n in enumerate(p.lens)]).contiguous()
    o, l = rect.window_attention_return_lse(p.q, p.kc.squeeze(1), p.vc.squeeze(1), p.qo, _i32(ph.offsets(p.lens)), kv_indices, 99, p.sm)
    out, lse = p.run(ext)
    _, _, to, tl = p.want()
    assert torch.all((out.double() - o.double()).abs() <= 2 * to) and torch.all((lse - l).double().abs() <= 2 * tl)


@pytest.mark.parametrize("rows", [1, 6, 90])
def test_a_query_that_is_not_finite_spares_the_others(ext, rows):
    p = Problem([rows, rows], [rows + 200, rows + 30], 8, 2, 128, 16)
    want = p.run(ext)
    p.q[rows // 2, 3, 5] = math.nan
    p.q[rows + rows // 3, 1] = math.inf
    out, lse = p.run(ext)
    hit = torch.zeros(2 * rows, 8, dtype=torch.bool, device=DEV)
    hit[rows // 2, 3] = hit[rows + rows // 3, 1] = True
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(out[~hit], want[0][~hit]) and torch.equal(lse[~hit], want[1][~hit])


@pytest.mark.parametrize("rows,hq", [(1, 4), (20, 16)])
def test_the_most_requests(ext, rows, hq):
    """4096 requests (decode, and tasks of 128 columns), checked on a sample."""
    new = [rows] * 4096
    lens = [rows + 7 * i % 50 for i in range(4096)]
    p = Problem(new, lens, hq, 2, 64, 4, seed=8)
    out, lse = p.run(ext)
    for b in (0, 1, 77, 2048, 4094, 4095):
        at = b * rows
        want = ph.attention(p.q[at:at + rows], p.k, p.v, [rows], [lens[b]], p.table[b:b + 1], 4, p.kc.shape[0], p.sm)
        ph.assert_close(out[at:at + rows], want[0], want[2], f"out of request {b}")
        ph.assert_close(lse[at:at + rows], want[1], want[3], f"lse of request {b}")
    with pytest.raises(RuntimeError, match="4096"):
        qo, kl = _i32([0] * 4098), _i32([1] * 4097)
        ext.mac_paged_chunk_attention(p.q, p.kc, p.vc, qo, kl, p.table[:1].expand(4097, -1), p.sm, kv_scales=p.sc)


def test_windows_past_the_table(ext):
    """Rows whose whole window lies past the keys that the table names."""
    p = Problem([2, 40, 1], [500, 300, 900], 4, 2, 64, 16, window=30)
    p.table = p.table[:, :10].contiguous()
    p.check(p.run(ext))


def test_a_window_wider_than_any_request(ext):
    p = Problem([5, 40], [300, 77], 8, 2, 128, 16)
    want = p.run(ext)
    for w in (299, 1 << 30, (1 << 31) - 1, 1 << 40):
        got = p.run(ext, window_left=w)
        if w >= 1 << 30:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        p.check(got)


def test_empty_batches(ext):
    p = Problem([1], [9], 2, 1, 64, 16)
    none = torch.empty(0, 2, 64, device=DEV, dtype=BF)
    for qo, lens in (([0], []), ([0, 0], [5])):
        out, lse = ext.mac_paged_chunk_attention(none, p.kc, p.vc, _i32(qo), _i32(lens), p.table, p.sm, kv_scales=p.sc)
        assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    # a table without columns: no keys
    out, lse = ext.mac_paged_chunk_attention(p.q, p.kc, p.vc, p.qo, p.kv_lens, p.table[:, :0], p.sm, kv_scales=p.sc)
    assert torch.all(out == 0) and torch.all(lse == -math.inf)


def test_refusals(ext):
    p = Problem([2, 1], [40, 20], 8, 2, 128, 16)

    def refused(text, **kw):
        a = dict(q=p.q, k_cache=p.kc, v_cache=p.vc, qo_indptr=p.qo, kv_lens=p.kv_lens, page_table=p.table, sm_scale=p.sm,
                 kv_scales=p.sc)
        a.update(kw)
        with pytest.raises(RuntimeError, match=text):
            ext.mac_paged_chunk_attention(**a)

    refused("bfloat16 or float16", q=p.q.float())
    refused("must be CUDA", q=p.q.cpu())
    refused("wrong shape", q=p.q[..., :64])
    refused("multiple of Hkv", q=p.q[:, :7])
    refused("must be float8_e4m3fn", k_cache=p.kc.float(), v_cache=p.vc.float(), kv_scales=None)
    refused("of q's dtype", k_cache=p.kc.half(), v_cache=p.vc.half(), kv_scales=None)
    refused("kv_scales belong", k_cache=p.kc.to(BF), v_cache=p.vc.to(BF))
    refused("head_dim must be", q=p.q[..., :96], k_cache=p.kc[..., :96], v_cache=p.vc[..., :96], kv_scales=p.sc)
    refused("wrong dtype", qo_indptr=p.qo.long())
    refused("wrong length", kv_lens=p.kv_lens[:1])
    refused("wrong length", req_ids=_i32([0]))
    refused("int32", page_table=p.table.long())
    refused("fewer rows", page_table=p.table[:1])
    refused("contiguous rows", page_table=p.table.t().contiguous().t())
    refused("sm_scale", sm_scale=0.0)
    refused("sm_scale", sm_scale=float("inf"))
    refused("logit_cap", logit_cap=-1.0)
    refused("does not fit fp32", sm_scale=1e-60)
    refused("does not fit fp32", logit_cap=1e300)
    refused("takes no k_scale", k_scale=0.5)
    refused("positive", kv_scales=None, v_scale=-1.0)
    refused("out must be", out=torch.empty(3, 8, 64, device=DEV, dtype=BF))
    refused("out_lse must be", out_lse=torch.empty(3, 8, device=DEV, dtype=BF))
    refused("same strides", k_cache=p.kc, v_cache=p.vc.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(ph.F8))
    refused("positive", kv_scales=None, k_scale=1e300)
    refused("out of range", window_left=-(1 << 40))
    refused("power of two", k_cache=p.kc[:, :12], v_cache=p.vc[:, :12], kv_scales=None)
