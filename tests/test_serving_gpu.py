"""The serving entry points on the GPU against plain implementations in 64 bits: the quantised cache written and read back,
attention over its pages and over a shared prefix, the gated delta rule with a carried state, and a run of them together.

Tolerances.  A result rounded to bf16 is off by at most 2^-8 of its value (half a step).  Attention adds the rounding of each
weight to f16 (2^-11 of it, 2^-25 of the largest below f16's normal range) and the error of the scores: a dot product of D
terms in fp32 is off by at most D * 2^-24 of the sum of its terms' magnitudes, which moves a weight by that part of itself, in the
sum and in the product.  The delta rule's bound is carried along with the recurrence (`delta_ref`)."""
import itertools
import math

import pytest
import torch

from reax_engine_kernels_b200 import kernels as rk
from reax_engine_kernels_b200 import synth

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def status():
    return rk.status("libreax_decode")


@pytest.fixture(autouse=True)
def clear_status():
    status()
    yield
    assert status() == 0, "a kernel reported something that the test did not expect"


# ------------------------------------------------------------------------------------------------ the cache
def e4m3_values():
    out = []
    for b in range(127):
        e, m = b >> 3, b & 7
        out.append(math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10))
    return torch.tensor(out, dtype=torch.float64)


def quantise_ref(x):
    """[..., D] -> (bytes, exponent bytes) in 64 bits, by search in the table of the 127 nonnegative values."""
    x = x.double().cpu()
    amax = x.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    n = torch.full(amax.shape, -127)
    for i in itertools.product(*map(range, amax.shape)):
        if not bad[i] and amax[i] > 0:
            k = -127
            while amax[i].item() > math.ldexp(448.0, k):
                k += 1
            n[i] = k
    y = torch.where(bad[..., None], 0.0, x) / torch.pow(2.0, n.double())[..., None]
    tab = e4m3_values()
    hi = torch.searchsorted(tab, y.abs().contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = y.abs() - tab[lo], tab[hi] - y.abs()
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = code | torch.where(torch.signbit(y), 128, 0)
    return code.to(torch.uint8), torch.where(bad, 255, n + 127).to(torch.uint8)


def value_ref(code, e):
    """64-bit values of bytes and exponent bytes."""
    tab = torch.cat([e4m3_values(), torch.tensor([math.nan], dtype=torch.float64)])
    tab = torch.cat([tab, -tab]).to(code.device)
    return tab[code.long()] * torch.where(e == 255, math.nan, torch.pow(2.0, e.double() - 127))[..., None]


def odd_rows(g, T, H, D):
    """Rows of all magnitudes, zeros, ties, values next to a power of two's border, subnormals, infinities, NaN."""
    x = (randn(g, T, H, D) * torch.exp(3 * randn(g, T, H, 1))).to(BF)
    f = x.view(T * H, D)
    special = [torch.zeros(D), torch.full((D,), 448.0), torch.full((D,), 450.0), torch.full((D,), 1e-40), torch.full((D,), 2.0 ** -126),
               torch.full((D,), 3.3e38), torch.full((D,), -0.0), torch.arange(D) / 16.0 + 1 / 32]
    for i, s in enumerate(special):
        if i < f.shape[0]:
            f[i] = s.to(DEV).to(BF)
    if f.shape[0] > 12:
        f[9, 3], f[10, D - 1], f[11, 0] = math.inf, math.nan, -math.inf
    return x


@pytest.mark.parametrize("T,H,D,page", [(1, 1, 128, 16), (7, 3, 128, 48), (33, 2, 256, 16), (130, 4, 128, 64), (1500, 8, 256, 32)])
@pytest.mark.parametrize("fused", [False, True])
def test_cache_written_and_read(T, H, D, page, fused):
    g = gen(T + D)
    pages = T // page + 3
    if fused:  # k and v as slices of a projection's rows, both caches in one allocation
        row = torch.zeros(T, 2 * H * D + 8, dtype=BF, device=DEV)
        k, v = row[:, 8:8 + H * D].view(T, H, D), row[:, 8 + H * D:].view(T, H, D)
        k.copy_(odd_rows(g, T, H, D))
        v.copy_(odd_rows(g, T, H, D))
        kv = torch.full((pages, 2, H, page, D), 0x5A, dtype=torch.uint8, device=DEV)
        e = torch.full((pages, 2, H, page), 77, dtype=torch.uint8, device=DEV)
        c = rk.KvCache(kv[:, 0].view(torch.float8_e4m3fn), e[:, 0], kv[:, 1].view(torch.float8_e4m3fn), e[:, 1])
    else:
        k, v = odd_rows(g, T, H, D), odd_rows(g, T, H, D).flip(-1)
        c = rk.kv_cache(pages, H, page, D)
        for t in c:
            t.view(torch.uint8).fill_(0x5A)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:T].contiguous()
    if T > 1:
        slots[T // 2] = -1
    was = [t.view(torch.uint8).clone() for t in c]
    rk.kv_write(k, v, c, slots)
    live = slots >= 0
    at = slots[live]
    pg, off = at // page, at % page
    for x, code, e, code0, e0 in ((k, c.k, c.ke, was[0], was[1]), (v, c.v, c.ve, was[2], was[3])):
        wc, we = quantise_ref(x[live])
        assert torch.equal(code.view(torch.uint8)[pg, :, off].cpu(), wc)
        assert torch.equal(e[pg, :, off].cpu(), we)
        # nothing else was written
        code0[pg, :, off], e0[pg, :, off] = wc.to(DEV), we.to(DEV)
        assert torch.equal(code.view(torch.uint8), code0) and torch.equal(e, e0)
    rkk, rvv = rk.kv_read(c, slots)
    for got, x in ((rkk, k), (rvv, v)):
        wc, we = quantise_ref(x)
        want = value_ref(wc, we).to(torch.float32).to(BF).to(DEV)
        want[~live] = 0
        assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))


def test_large_write_two_rows_a_thread():
    """Past ten waves of CTAs a thread writes two rows: the same codes as in parts that do not reach it."""
    T, H, D, page = 12501 * torch.cuda.get_device_properties(0).multi_processor_count // 148, 8, 256, 16
    g = gen(77)
    k, v = randn(g, T, H, D).to(BF), odd_rows(g, T, H, D)
    slots = torch.randperm(-(-T // page) * page, generator=g, device=DEV)[:T].contiguous()
    slots[T // 3] = -1
    a, b = (rk.kv_cache(-(-T // page), H, page, D) for _ in range(2))
    rk.kv_write(k, v, a, slots)
    for i in range(0, T, 1000):
        rk.kv_write(k[i:i + 1000], v[i:i + 1000], b, slots[i:i + 1000])
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    wc, we = quantise_ref(v[-50:])
    at = slots[-50:]
    assert torch.equal(a.v.view(torch.uint8)[at // page, :, at % page].cpu(), wc) and torch.equal(a.ve[at // page, :, at % page].cpu(), we)


def test_slots_past_the_end_are_skipped_and_reported():
    g = gen(5)
    k = randn(g, 4, 2, 128).to(BF)
    c = rk.kv_cache(2, 2, 16, 128)
    s = torch.tensor([3, 32, 1 << 40, 31], device=DEV)
    rk.kv_write(k, k, c, s)
    assert status() == 0x501
    n = c.ke.count_nonzero().item()
    assert n == 2 * 2
    a, b = rk.kv_read(c, s)
    assert status() == 0x501
    assert a[1:3].count_nonzero() == 0 and a[0].count_nonzero() > 0 and torch.equal(a, b)


def test_empty_calls():
    c = rk.kv_cache(2, 2, 16, 128)
    z = torch.zeros(0, 2, 128, dtype=BF, device=DEV)
    rk.kv_write(z, z, c, torch.zeros(0, dtype=torch.int64, device=DEV))
    a, b = rk.kv_read(c, torch.zeros(0, dtype=torch.int64, device=DEV))
    assert a.shape == b.shape == (0, 2, 128)
    o = rk.fmha_paged(torch.zeros(0, 2, 4, 128, dtype=BF, device=DEV), c, torch.zeros(0, 2, dtype=torch.int32, device=DEV), 1.0,
                      qpos=torch.zeros(0, 4, dtype=torch.int32, device=DEV))
    assert o.shape == (0, 2, 4, 128)


def test_cache_past_32_bits():
    """Rows whose byte offset in the cache lies past 2^32."""
    pages, H, page, D = (1 << 32) // (8 * 64 * 256) + 2, 8, 64, 256
    k = torch.empty(pages, H, page, D, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    e = torch.zeros(pages, H, page, dtype=torch.uint8, device=DEV)
    c = rk.KvCache(k, e, k.clone(), e.clone())
    g = gen(9)
    x, y = randn(g, 40, H, D).to(BF), randn(g, 40, H, D).to(BF)
    s = torch.arange(40, device=DEV) + pages * page - 40
    rk.kv_write(x, y, c, s)
    a, b = rk.kv_read(c, s)
    assert (a - x).abs().max() <= x.abs().max() * 2 ** -4 and (b - y).abs().max() <= y.abs().max() * 2 ** -4
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=DEV)
    q = randn(g, 1, H, 1, D).to(BF)
    o = rk.fmha_paged(q, c, table, 0.1, qpos=torch.tensor([[63]], dtype=torch.int32, device=DEV))
    assert_attention(o, q, c, table, 0.1, torch.tensor([[63]], dtype=torch.int32, device=DEV), 1)


# ------------------------------------------------------------------------------------------------ attention
def filled(g, pages, H, page, D, spread=1.0):
    c = rk.kv_cache(pages, H, page, D)
    n = pages * page
    x, y = (randn(g, n, H, D) * torch.exp(spread * randn(g, n, H, 1)) for _ in range(2))
    rk.kv_write(x.to(BF), y.to(BF), c, torch.arange(n, device=DEV))
    return c


def assert_attention(o, q, c, table, scale, qpos, G, prefix=None, Lp=0, bad=()):
    """Each row against the formula in 64 bits, within the bound of this file's head."""
    B, H, M, D = q.shape
    page = c.k.shape[2]
    kc, vc = (t.view(torch.uint8) for t in (c.k, c.v))
    for b in range(B):
        pages = ([] if prefix is None else prefix.tolist())
        own = table[b].tolist()
        for r in range(M):
            last = int(qpos[b, r // G])
            n = min(last + 1, Lp + table.shape[1] * page)
            where = [(pages[j // page], j % page) if j < Lp else (own[(j - Lp) // page], (j - Lp) % page) for j in range(max(n, 0))]
            where = [w for w in where if w[0] not in bad]
            if not where:
                assert o[b, :, r].count_nonzero() == 0
                continue
            pg, off = (torch.tensor(x, device=DEV) for x in zip(*where))
            k, v = (value_ref(t[pg, :, off], e[pg, :, off]) for t, e in ((kc, c.ke), (vc, c.ve)))  # [n, H, D]
            qr = q[b, :, r].double()
            s = torch.einsum("hd,nhd->hn", qr, k) * scale
            size = torch.einsum("hd,nhd->hn", qr.abs(), k.abs()).amax(-1) * abs(scale)
            p = torch.softmax(s, -1)
            want = torch.einsum("hn,nhd->hd", p, v)
            mean = torch.einsum("hn,nhd->hd", p, v.abs())
            big = v.abs().amax((0, 2)) * len(where) * 2.0 ** -24  # below f16's normal range, and e4m3 rows reach 448 / 224 of it
            part = 2.0 ** -11 + 2 * (D + 8) * 2.0 ** -24 * size + 2.0 ** -18
            tol = 2.0 ** -8 * want.abs() + part[:, None] * mean * 1.01 + big[:, None]
            got = o[b, :, r].double()
            nan = torch.isnan(want)
            assert torch.equal(torch.isnan(got), nan), (b, r)
            off_by = ((got - want).abs() - tol)[~nan]
            assert off_by.numel() == 0 or off_by.max() <= 0, (b, r, off_by.max().item())


def setup(seed, B, H, G, Tq, D, page, lens, Lp=0, spread=1.0, extra=2):
    g = gen(seed)
    P, PP = max(1, max(-(-n // page) for n in lens)) + 1, -(-Lp // page)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + PP + extra
    c = filled(g, pages, H, page, D, spread)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, P), -5, dtype=torch.int32, device=DEV)  # entries behind a sequence's end are never followed
    at = PP
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    qpos = torch.tensor([[Lp + n - Tq + t for t in range(Tq)] for n in lens], dtype=torch.int32, device=DEV)
    q = randn(g, B, H, Tq * G, D).to(BF)
    return q, c, table, qpos, order[:PP].contiguous()


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("H,G,Tq,page,lens", [
    (1, 1, 1, 16, [1]),
    (2, 4, 1, 16, [1, 15, 16, 17]),
    (2, 8, 2, 32, [2, 63, 64, 65, 511]),
    (1, 5, 3, 48, [3, 100, 257]),          # 15 rows, a page size that is no power of two
    (2, 4, 8, 16, [8, 300]),               # 32 rows: two row tiles
    (1, 17, 1, 64, [700, 33]),             # 17 rows
    (3, 1, 4, 16, [4, 1023, 1025]),        # a late chunk of one key
    (8, 4, 1, 16, [5000]),                 # many chunks
])
def test_paged_attention(D, H, G, Tq, page, lens):
    q, c, table, qpos, _ = setup(len(lens) + D, len(lens), H, G, Tq, D, page, lens)
    o = rk.fmha_paged(q, c, table, D ** -0.5, qpos=qpos, G=G)
    assert_attention(o, q, c, table, D ** -0.5, qpos, G)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("H,G,Tq,page,lens,Lp", [
    (1, 1, 1, 16, [1, 2], 1),
    (2, 4, 1, 16, [1, 40, 16], 47),
    (2, 4, 2, 32, [2, 300, 7, 64, 65], 700),
    (1, 8, 3, 64, [3, 500], 1601),
    (1, 4, 1, 16, [20] * 40, 333),         # 160 rows on the prefix
    (2, 16, 1, 32, [40] * 9, 500),         # 144 rows: a second tile of 128 with 16
])
def test_shared_prefix(D, H, G, Tq, page, lens, Lp):
    q, c, table, qpos, prefix = setup(Lp + D, len(lens), H, G, Tq, D, page, lens, Lp)
    o = rk.fmha_paged(q, c, table, D ** -0.5, qpos=qpos, G=G, prefix=prefix, prefix_len=Lp)
    assert_attention(o, q, c, table, D ** -0.5, qpos, G, prefix, Lp)


@pytest.mark.parametrize("D", [128, 256])
def test_rows_that_see_part_of_the_prefix_or_nothing(D):
    q, c, table, qpos, prefix = setup(3, 6, 2, 2, 3, D, 16, [30] * 6, 100)
    qpos = torch.tensor([[-1, -1, -1], [-1, 0, 1], [50, 99, 100], [98, 16, 129], [128, 129, 1 << 30], [-(1 << 31), 2147483647, 5]],
                        dtype=torch.int32, device=DEV)
    # the table's last entry is out of range, and rows with a far qpos reach it
    table[:, 2:] = prefix[:1]
    o = rk.fmha_paged(q, c, table, 0.07, qpos=qpos, G=2, prefix=prefix, prefix_len=100)
    assert_attention(o, q, c, table, 0.07, qpos, 2, prefix, 100)
    o = rk.fmha_paged(q, c, table, 0.07, qpos=qpos, G=2)
    assert_attention(o, q, c, table, 0.07, qpos, 2)
    none = torch.zeros(6, 0, dtype=torch.int32, device=DEV)  # no pages of their own
    o = rk.fmha_paged(q, c, none, 0.07, qpos=qpos, G=2, prefix=prefix, prefix_len=100)
    assert_attention(o, q, c, none, 0.07, qpos, 2, prefix, 100)
    assert rk.fmha_paged(q, c, none, 0.07, qpos=qpos, G=2).count_nonzero() == 0


# G = 4 rows a sequence keep the prefix with the kernel for few rows, more take it to the one of 128-row tiles
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("G,Lp", [(4, 0), (4, 130), (8, 130), (50, 130)])
def test_masked_rows_may_hold_anything(G, Lp, D):
    """Bytes behind a sequence's end: NaN codes and NaN exponents, in its last page and in the prefix's."""
    lens = [5, 70, 16]
    q, c, table, qpos, prefix = setup(11, 3, 2, G, 1, D, 32, lens, Lp)
    for t in (c.k, c.v):
        u = t.view(torch.uint8)
        for b, n in enumerate(lens):
            if n % 32:
                u[table[b, n // 32].long(), :, n % 32:] = 0x7F
        if Lp:
            u[prefix[-1].long(), :, Lp % 32:] = 0xFF
    for t in (c.ke, c.ve):
        for b, n in enumerate(lens):
            if n % 32:
                t[table[b, n // 32].long(), :, n % 32:] = 255
        if Lp:
            t[prefix[-1].long(), :, Lp % 32:] = 255
    o = rk.fmha_paged(q, c, table, 0.1, qpos=qpos, G=G, prefix=prefix if Lp else None, prefix_len=Lp)
    assert torch.isfinite(o).all()
    assert_attention(o, q, c, table, 0.1, qpos, G, prefix if Lp else None, Lp)


@pytest.mark.parametrize("G,Lp", [(2, 0), (2, 100), (4, 100)])
def test_nan_rows_reach_only_the_queries_that_see_them(G, Lp):
    """A NaN key (or value) row among a sequence's new tokens: queries before it are finite, the others NaN."""
    q, c, table, qpos, prefix = setup(12, 2, 1, G, 4, 128, 16, [40, 41], Lp)
    p, off = table[0, 38 // 16].long(), 38 % 16
    c.ke[p, 0, off] = 255
    p, off = table[1, 40 // 16].long(), 40 % 16
    c.ve[p, 0, off] = 255
    o = rk.fmha_paged(q, c, table, 0.1, qpos=qpos, G=G, prefix=prefix if Lp else None, prefix_len=Lp)
    assert_attention(o, q, c, table, 0.1, qpos, G, prefix if Lp else None, Lp)


@pytest.mark.parametrize("G", [2, 4])
@pytest.mark.parametrize("D", [128, 256])
def test_nan_rows_in_the_prefix(G, D):
    """A NaN key row, and a NaN value row, of the prefix: only rows whose qpos lies before them are finite."""
    for which in ("ke", "ve"):
        q, c, table, qpos, prefix = setup(33, 2, 1, G, 4, D, 16, [40, 41], 150)
        getattr(c, which)[prefix[99 // 16].long(), 0, 99 % 16] = 255
        qpos[0] = torch.tensor([20, 98, 99, 149], dtype=torch.int32)
        o = rk.fmha_paged(q, c, table, 0.1, qpos=qpos, G=G, prefix=prefix, prefix_len=150)
        assert torch.isfinite(o[0, :, :2 * G]).all() and torch.isnan(o[0, :, 2 * G:]).all() and torch.isnan(o[1]).all()
        assert_attention(o, q, c, table, 0.1, qpos, G, prefix, 150)


@pytest.mark.parametrize("G", [3, 8])
def test_far_magnitudes(G):
    """Queries and rows of very different powers of two, a scale below zero, an outlier channel."""
    for D, scale, spread in ((128, 0.1, 4.0), (256, -0.05, 2.0), (128, 1e-3, 8.0)):
        q, c, table, qpos, prefix = setup(13 + D, 3, 2, G, 1, D, 16, [50, 200, 333], 90, spread)
        q[0] *= 1e-20
        q[1, :, :, 5] *= 300
        q[2] *= 2.0 ** 20
        sc = scale if spread < 8 else scale * 1e-3
        q[2] *= 2.0 ** -18
        o = rk.fmha_paged(q, c, table, sc, qpos=qpos, G=G, prefix=prefix, prefix_len=90)
        assert_attention(o, q, c, table, sc, qpos, G, prefix, 90)


@pytest.mark.parametrize("G,Lp", [(2, 0), (2, 64), (20, 64)])
def test_page_ids_out_of_range_are_not_seen_and_reported(G, Lp):
    q, c, table, qpos, prefix = setup(14, 2, 2, G, 1, 128, 32, [100, 90], Lp)
    n = c.k.shape[0]
    table[0, 1], table[1, 0] = n, -1
    if Lp:
        prefix[1] = 1 << 30
    o = rk.fmha_paged(q, c, table, 0.1, qpos=qpos, G=G, prefix=prefix if Lp else None, prefix_len=Lp)
    assert status() == 0x502
    assert_attention(o, q, c, table, 0.1, qpos, G, prefix if Lp else None, Lp, bad=(n, -1, 1 << 30))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("page,Lp", [(16, 1001), (48, 700), (64, 1000), (96, 1001), (128, 129), (192, 1151), (256, 1)])
def test_prefix_in_pages_of_every_kind(page, Lp, D):
    """A tile of 64 prefix keys comes in as many rows at a time as surely lie in one page: 16, 32 or 64.  One page of several is
    missing; the tiles outnumber the buffers in flight."""
    q, c, table, qpos, prefix = setup(41, 5, 2, 8, 1, D, page, [3, 70, 1, 33, 12], Lp)
    bad = ()
    if len(prefix) > 2:
        prefix[1] = bad_id = c.k.shape[0] + 7
        bad = (bad_id,)
    o = rk.fmha_paged(q, c, table, D ** -0.5, qpos=qpos, G=8, prefix=prefix, prefix_len=Lp)
    assert status() == (0x502 if bad else 0)
    assert_attention(o, q, c, table, D ** -0.5, qpos, 8, prefix, Lp, bad=bad)


def test_long_prefix_wraps_the_buffers():
    """Few heads and a long prefix, so that a CTA's tiles go around its buffers many times; bits equal on a second run."""
    for D in (128, 256):
        q, c, table, qpos, prefix = setup(43, 5, 1, 8, 1, D, 64, [3, 70, 1, 33, 12], 64 * 64 * 20 - 5)
        o, o2 = (rk.fmha_paged(q, c, table, D ** -0.5, qpos=qpos, G=8, prefix=prefix, prefix_len=64 * 64 * 20 - 5) for _ in range(2))
        assert status() == 0 and torch.equal(o, o2)
        rows = slice(0, 2)
        assert_attention(o[rows], q[rows], c, table[rows], D ** -0.5, qpos[rows], 8, prefix, 64 * 64 * 20 - 5)


def test_strided_operands():
    """q and out as [B, Tq, Hq, D] tensors of wider rows, folded by strides; qpos and table as slices."""
    B, H, G, Tq, D = 3, 2, 4, 2, 128
    q, c, table, qpos, prefix = setup(15, B, H, G, Tq, D, 16, [20, 33, 700], 50)
    wide = torch.full((B, Tq, H * G, D + 8), 7.0, dtype=BF, device=DEV)
    owide = torch.full((B, Tq, H * G, D + 16), 7.0, dtype=BF, device=DEV)
    for t in range(Tq):  # one token at a time: row r = query head, stride D + 8
        qt = wide[:, t].view(B, H, G, D + 8)[..., :D]
        qt.copy_(q.view(B, H, Tq, G, D)[:, :, t])
        ot = owide[:, t].view(B, H, G, D + 16)[..., :D]
        qp = torch.stack([qpos[:, t]] * 3, 1)[:, 1:]
        tb = torch.cat([table, table], 1)[:, :table.shape[1]]
        rk.fmha_paged(qt, c, tb, 0.1, qpos=qp, G=G, prefix=prefix, prefix_len=50, out=ot)
        assert_attention(ot, qt, c, table, 0.1, qpos[:, t:t + 1], G, prefix, 50)
    assert (owide[..., D:] == 7).all()


def test_graph_replays_with_other_lengths_and_two_graphs_share_nothing():
    lens = [400, 30, 7]
    q, c, table, qpos, prefix = setup(16, 3, 2, 4, 1, 256, 16, lens, 200)
    outs, graphs = [], []
    for Lp in (0, 200):
        kw = dict(qpos=qpos, G=4, prefix=prefix if Lp else None, prefix_len=Lp)
        rk.fmha_paged(q, c, table, 0.1, **kw)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = rk.fmha_paged(q, c, table, 0.1, **kw)
        outs.append(o)
        graphs.append(gr)
    for cut in ([0, 0, 0], [390, 29, 0], [399, 1, 7]):
        qpos.copy_(torch.tensor([[200 + n - 1 - x] for n, x in zip(lens, cut)], dtype=torch.int32))
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert_attention(outs[1], q, c, table, 0.1, qpos, 4, prefix, 200)
        # without the prefix these positions reach past a history's pages, to entries of -5: reported, not seen
        assert_attention(outs[0], q, c, table, 0.1, qpos, 4, bad=(-5,))
    status()


@pytest.mark.parametrize("captured", [False, True])
def test_inputs_made_on_another_stream(captured):
    """The kernels start as dependents of what their stream holds before them: what another stream made, joined by an event, is
    waited for all the same, and so is the consumer on a third stream for them."""
    B, H, G, D, page, L = 3, 2, 4, 128, 16, 200
    q0, c, table, qpos, prefix = setup(31, B, H, G, 1, D, page, [L] * B, 100)
    g = gen(32)
    k0, v0 = randn(g, B, H, D).to(BF), randn(g, B, H, D).to(BF)
    slots = table.long()[torch.arange(B, device=DEV), (L - 1) // page] * page + (L - 1) % page
    d = delta_inputs(33, [1, 40, 16], 2, 4, 3)
    st0 = d["state"].clone()
    q, k, v, dk = (torch.zeros_like(x) for x in (q0, k0, v0, d["k"]))
    big = torch.randn(4096, 4096, device=DEV)
    out = {}

    def run():
        main, s1, s2 = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()
        s1.wait_stream(main)
        with torch.cuda.stream(s1):  # a producer that takes a while
            x = big
            for _ in range(6):
                x = x @ big * 1e-2
            for dst, src in ((q, q0), (k, k0), (v, v0), (dk, d["k"])):
                dst.copy_(src)
            d["state"].copy_(st0)
        scratch = big[0] * 2  # a kernel of this stream's own just before the join
        main.wait_stream(s1)
        rk.kv_write(k, v, c, slots)
        o = rk.fmha_paged(q, c, table, D ** -0.5, qpos=qpos, G=G, prefix=prefix, prefix_len=100)
        r = rk.delta_state(d["q"], dk, d["v"], d["g"], d["beta"], d["cu"], 0.1, d["state"])
        s2.wait_stream(main)
        with torch.cuda.stream(s2):
            out["o"], out["r"] = o.clone(), r.clone()
        main.wait_stream(s2)
        out["keep"] = (x, scratch, o, r)

    if captured:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
    for _ in range(3):
        for x in (q, k, v, dk):
            x.zero_()
        torch.cuda.synchronize()
        graph.replay() if captured else run()
        torch.cuda.synchronize()
        state = d["state"].clone()
        rk.kv_write(k0, v0, c, slots)
        o = rk.fmha_paged(q0, c, table, D ** -0.5, qpos=qpos, G=G, prefix=prefix, prefix_len=100)
        d["state"].copy_(st0)
        r = rk.delta_state(d["q"], d["k"], d["v"], d["g"], d["beta"], d["cu"], 0.1, d["state"])
        assert torch.equal(out["o"], o) and torch.equal(out["r"], r) and torch.equal(state, d["state"])


def test_same_bits_every_time():
    q, c, table, qpos, prefix = setup(17, 4, 2, 4, 1, 128, 16, [3000, 5, 900, 1], 600)
    a = [rk.fmha_paged(q, c, table, 0.1, qpos=qpos, G=4, prefix=prefix, prefix_len=600) for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


# ------------------------------------------------------------------------------------------------ delta rule
def delta_inputs(seed, lens, H, HV, S, decay=2.0, behind=0):
    g = gen(seed)
    T = sum(lens) + behind
    silu = torch.nn.functional.silu
    unit = lambda x: (x / x.square().sum(-1, keepdim=True).sqrt()).to(BF)  # noqa: E731
    cu = torch.tensor([0] + list(itertools.accumulate(lens)), dtype=torch.int64, device=DEV)
    return dict(q=unit(silu(randn(g, T, H, 128))), k=unit(silu(randn(g, T, H, 128))), v=randn(g, T, HV, 128).to(BF),
                g=-torch.nn.functional.softplus(randn(g, T, HV) - decay) * 1.4426950408889634,
                beta=torch.sigmoid(randn(g, T, HV)).to(BF), cu=cu, state=randn(g, S, HV, 128, 128))


def delta_ref(d, scale, slots=None, fresh=None):
    """The recurrence token by token in 64 bits, with a bound on what fp32 may add to each row of h (in its 2-norm).

    With |k| <= 1 + 2^-8 and beta <= 1 the map h -> 2^g (h - beta (h k) k^T) does not lengthen a row, so a row's error only
    decays, and a token adds at most c * 2^-24 * (2^g |h| + |v|): the dot product of 128 terms (128), its subtraction, products
    and the update (8), twice (h k enters the update through k), and exp2's 2 ulps."""
    q, k, v, beta, g = (d[n].double() for n in ("q", "k", "v", "beta", "g"))
    rep = v.shape[1] // q.shape[1]
    state = d["state"].double().clone()
    o, tol = torch.zeros_like(v), torch.zeros_like(v)
    btol = torch.zeros(state.shape[:3], dtype=torch.float64, device=DEV)
    cu = d["cu"].tolist()
    c = (2 * (128 + 8) + 4) * 2.0 ** -24
    for n in range(len(cu) - 1):
        s = n if slots is None else int(slots[n])
        if cu[n] == cu[n + 1] or s < 0:
            continue
        h = torch.zeros_like(state[s]) if fresh is not None and fresh[n] else state[s]
        e = torch.zeros_like(btol[s])
        for t in range(cu[n], cu[n + 1]):
            kt, qt = (x[t].repeat_interleave(rep, 0)[..., None] for x in (k, q))
            a = torch.exp2(g[t])[:, None]
            h = h * a[..., None]
            u = beta[t][:, None] * (v[t] - (h @ kt)[..., 0])
            e = e * a + c * (h.norm(dim=-1) + v[t].abs())
            h = h + u[..., None] * kt.transpose(-1, -2)
            o[t] = scale * (h @ qt)[..., 0]
            qn = qt[..., 0].norm(dim=-1)[:, None]
            tol[t] = 2.0 ** -8 * o[t].abs() + abs(scale) * qn * (e + c * h.norm(dim=-1)) * 1.01
        state[s], btol[s] = h, e
    return o, tol, state, btol


def assert_delta(d, scale, o, state0, live, slots=None, fresh=None):
    wo, tol, ws, wtol = delta_ref({**d, "state": state0}, scale, slots, fresh)
    assert ((o.double() - wo).abs() - tol)[live].max() <= 0
    off = (d["state"].double() - ws).norm(dim=-1)
    assert (off - wtol * 1.01).max() <= 0, (off.max().item(), wtol.max().item())


@pytest.mark.parametrize("H,HV,lens", [
    (1, 1, [1]), (2, 4, [1, 1, 1]), (4, 4, [2, 0, 3]), (1, 4, [5, 17, 1, 16]), (2, 6, [64, 1, 33]), (16, 32, [1] * 9),
    (2, 4, [200, 129]), (1, 2, [1000]), (2, 2, [8, 9, 31, 0, 32, 1, 33]), (1, 3, [65, 2, 96, 95]),
])
@pytest.mark.parametrize("fresh", [False, True])
def test_delta_state(H, HV, lens, fresh):
    d = delta_inputs(sum(lens) + HV, lens, H, HV, len(lens) + 2, behind=3)
    n = len(lens)
    slots = torch.randperm(n + 2, generator=gen(n), device=DEV)[:n].to(torch.int32)
    f = (torch.arange(n, device=DEV) % 2 == 0) if fresh else None
    if fresh:  # what a fresh sequence's slot holds is not read
        d["state"][slots[::2].long()] = math.nan
    state0 = d["state"].clone()
    if fresh:
        state0[slots[::2].long()] = 0
        for i in range(0, n, 2):
            if not lens[i]:
                d["state"][slots[i].long()] = 0
    T = d["q"].shape[0]
    o = torch.full((T, HV, 128), 7.0, dtype=BF, device=DEV)
    rk.delta_state(d["q"], d["k"], d["v"], d["g"], d["beta"], d["cu"], 0.088, d["state"], slots=slots, fresh=f, o=o)
    live = torch.arange(T, device=DEV) < sum(lens)
    assert (o[~live] == 7).all()
    assert_delta(d, 0.088, o, state0, live, slots, f)


def test_delta_state_decays_to_nothing_and_not_at_all():
    d = delta_inputs(3, [40, 40], 2, 4, 2)
    d["g"][:40, 0] = 0.0           # no decay
    d["g"][5, 1] = -math.inf       # forgets everything
    d["g"][7, 2] = -200.0
    d["g"][40:] = -30.0            # each token nearly forgets
    d["beta"][:, 3] = 0.0          # never learns
    d["beta"][:, 2] = 1.0
    state0 = d["state"].clone()
    o = rk.delta_state(*(d[n] for n in ("q", "k", "v", "g", "beta", "cu")), 1.0, d["state"])
    assert_delta(d, 1.0, o, state0, slice(None))


def test_delta_state_alike_keys():
    """All keys the same and beta 1: within a chunk every token overwrites what the one before it wrote."""
    d = delta_inputs(4, [100], 1, 2, 1)
    d["k"][:] = d["k"][:1]
    d["beta"][:] = 1.0
    d["g"][:] = 0.0
    state0 = d["state"].clone()
    o = rk.delta_state(*(d[n] for n in ("q", "k", "v", "g", "beta", "cu")), 1.0, d["state"])
    assert_delta(d, 1.0, o, state0, slice(None))


def test_delta_state_in_parts():
    """A prompt in two calls, then token by token, against one call over all of it."""
    d = delta_inputs(6, [150], 2, 4, 1)
    args = [d[n] for n in ("q", "k", "v", "g", "beta")]
    whole = d["state"].clone()
    o = rk.delta_state(*args, d["cu"], 0.1, whole)
    parts = []
    for a, b in [(0, 70), (70, 140)] + [(i, i + 1) for i in range(140, 150)]:
        parts.append(rk.delta_state(*(x[a:b] for x in args), torch.tensor([0, b - a], device=DEV), 0.1, d["state"]))
    got = torch.cat(parts)
    _, tol, _, wtol = delta_ref({**d, "state": delta_inputs(6, [150], 2, 4, 1)["state"]}, 0.1)
    assert ((got.double() - o.double()).abs() - 2 * tol).max() <= 0
    assert ((d["state"].double() - whole.double()).norm(dim=-1) - 2 * wtol).max() <= 0


def test_delta_state_slots():
    """Strided slots; a negative slot is left alone, one past the end and one named twice get NaN rows and are reported."""
    lens = [2, 1, 3, 1, 0, 2]
    d = delta_inputs(7, lens, 2, 4, 6)
    pool = torch.full((6, 5, 128, 128), 3.0, device=DEV)[:, :4]
    pool.copy_(d["state"])
    d["state"] = pool
    state0 = pool.clone()
    slots = torch.tensor([3, -1, 6, 3, 0, 0], dtype=torch.int32, device=DEV)
    o = torch.full((9, 4, 128), 7.0, dtype=BF, device=DEV)
    rk.delta_state(*(d[n] for n in ("q", "k", "v", "g", "beta", "cu")), 1.0, pool, slots=slots, o=o)
    assert status() == 0x503
    assert (o[2] == 7).all() and torch.isnan(o[3:7]).all()
    live = torch.tensor([0, 1, 7, 8], device=DEV)
    ref = torch.tensor([3, -1, -1, -1, -1, 0], dtype=torch.int32, device=DEV)
    assert_delta(d, 1.0, o, state0, live, ref)


def test_delta_state_as_the_chunked_kernels():
    """A prompt from a zero state: reax_kkt + reax_howu round to bf16 at eight points of a chunk (operands kb, vb, the inverse A, u, w,
    vn, vdec and the state), each by at most 2^-8, so the two agree in the 2-norm within eight of them."""
    lens = [256, 100]
    s = synth.delta_rule_inputs(lens, 2, 4, 77)
    T_ = synth.to_torch_bf16
    q, k, v, beta, A = T_(s["q"]), T_(s["k"]), T_(s["v"]), T_(s["beta"]), None
    gc, cu, cidx = (torch.from_numpy(s[n]).cuda() for n in ("g", "cu", "cidx"))
    A = rk.kkt(k, gc, beta, cu, cidx, 4)
    want = rk.howu(q, k, v, beta, A, gc, cu, 0.0884)
    per = gc.clone()  # the token's own decay out of the chunk-local sums
    for a, b in zip(s["cu"][:-1], s["cu"][1:]):
        for c in range(a, b, 64):
            per[c + 1:min(c + 64, b)] -= gc[c:min(c + 64, b) - 1]
    state = torch.full((2, 4, 128, 128), math.nan, device=DEV)
    got = rk.delta_state(q, k, v, per, beta, cu, 0.0884, state, fresh=torch.ones(2, dtype=torch.bool, device=DEV))
    assert (got.double() - want.double()).norm() <= 8 * 2.0 ** -8 * want.double().norm()
    assert torch.isfinite(state).all()


def test_delta_state_short_sequence_and_rows_behind_it():
    """One sequence that is much shorter than the rows there are; T = N with uneven lengths."""
    for lens, behind in (([3], 60), ([50, 0, 0, 1] + [0] * 47, 0)):
        d = delta_inputs(31, lens, 1, 2, len(lens), behind=behind)
        state0 = d["state"].clone()
        o = torch.full((sum(lens) + behind, 2, 128), 7.0, dtype=BF, device=DEV)
        rk.delta_state(*(d[n] for n in ("q", "k", "v", "g", "beta", "cu")), 0.3, d["state"], o=o)
        assert (o[sum(lens):] == 7).all()
        assert_delta(d, 0.3, o, state0, slice(0, sum(lens)))


def test_delta_state_sequences_do_not_reach_each_other():
    """NaN inputs of one sequence, and of the rows behind the last one, stay there."""
    lens = [40, 5, 70, 3]
    d = delta_inputs(32, lens, 2, 4, 4, behind=4)
    clean = {n: t.clone() for n, t in d.items()}
    for n in ("q", "k", "v", "g", "beta"):
        d[n][40:45] = math.nan
        d[n][118:] = math.nan
    state0 = d["state"].clone()
    o = rk.delta_state(*(d[n] for n in ("q", "k", "v", "g", "beta", "cu")), 1.0, d["state"])
    assert torch.isnan(d["state"][1]).all()
    d["state"][1] = delta_ref({**clean, "state": state0}, 1.0)[2][1].float()
    live = torch.tensor([t for t in range(118) if not 40 <= t < 45], device=DEV)
    assert_delta({**clean, "state": d["state"]}, 1.0, o, state0, live)


def test_delta_state_graph_and_streams():
    d = delta_inputs(8, [1] * 5, 2, 4, 5)
    args = [d[n] for n in ("q", "k", "v", "g", "beta", "cu")]
    start = d["state"].clone()
    rk.delta_state(*args, 1.0, d["state"])
    d["state"].copy_(start)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        o = rk.delta_state(*args, 1.0, d["state"])
    d["state"].copy_(start)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        gr.replay()
        gr.replay()
    torch.cuda.synchronize()
    ref = start.clone()
    for _ in range(2):
        want = rk.delta_state(*args, 1.0, ref)
    assert torch.equal(o, want) and torch.equal(ref, d["state"])


# ------------------------------------------------------------------------------------------------ together
def test_serving_run():
    """A prompt and two steps of the two layer kinds.  Attention: the prompt's rows are quantised, read back for the prefill
    kernel, and each step writes its token and attends over the pages.  Linear attention: conv from the projection, the
    prompt's state by delta_state, each step's token through the conv cache and delta_state."""
    g = gen(21)
    H, G, D, page, L, steps = 2, 4, 128, 16, 77, 2
    c = rk.kv_cache(8, H, page, D)
    table = torch.tensor([[5, 2, 7, 0, 3, 6]], dtype=torch.int32, device=DEV)
    pos = torch.arange(L + steps, device=DEV)
    slots = table[0].long()[pos // page] * page + pos % page
    k, v = (randn(g, L + steps, H, D).to(BF) for _ in range(2))
    q = randn(g, L + steps, H * G, D).to(BF)
    rk.kv_write(k[:L], v[:L], c, slots[:L])
    kr, vr = rk.kv_read(c, slots[:L])
    # prefill over what the cache holds: row r = token r / G
    fold = q[:L].view(L, H, G, D).permute(1, 0, 2, 3).reshape(1, H, L * G, D)
    qp = torch.arange(L, dtype=torch.int32, device=DEV)[None]
    pre = rk.fmha(fold, kr.permute(1, 0, 2)[None], vr.permute(1, 0, 2)[None], D ** -0.5, qpos=qp, G=G)
    own = rk.fmha_paged(fold, c, table, D ** -0.5, qpos=qp, G=G)
    assert (pre.double() - own.double()).norm() <= 2.0 ** -7 * own.double().norm()  # each rounds p (2^-8 there) and o
    assert_attention(own[:, :, -2 * G:], fold[:, :, -2 * G:], c, table, D ** -0.5, qp[:, -2:], G)
    for t in range(L, L + steps):
        rk.kv_write(k[t:t + 1], v[t:t + 1], c, slots[t:t + 1])
        qt = q[t:t + 1].view(1, H, G, D)
        qp = torch.tensor([[t]], dtype=torch.int32, device=DEV)
        assert_attention(rk.fmha_paged(qt, c, table, D ** -0.5, qpos=qp, G=G), qt, c, table, D ** -0.5, qp, G)

    # linear attention: 2 key heads, 4 value heads of 128
    KD, VD = 256, 512
    SX = 2 * KD + VD
    x = randn(g, L + steps, SX).to(BF)
    w = (randn(g, SX, 4) * 0.5).to(BF)
    meta = torch.tensor([[i, 0, 0, 0] for i in range(L + steps)], dtype=torch.int32, device=DEV)
    allq, allk, allv = rk.conv_l2(x, meta, w, KD, VD)
    beta = torch.sigmoid(randn(g, L + steps, 4)).to(BF)
    gg = -torch.nn.functional.softplus(randn(g, L + steps, 4))
    state = torch.zeros(2, 4, 128, 128, device=DEV)
    heads = lambda a, n: a.view(-1, n, 128)  # noqa: E731
    slot = torch.tensor([1], dtype=torch.int32, device=DEV)
    cu = lambda n: torch.tensor([0, n], device=DEV)  # noqa: E731
    outs = [rk.delta_state(heads(allq[:L], 2), heads(allk[:L], 2), heads(allv[:L], 4), gg[:L], beta[:L], cu(L), 0.088, state,
                           slots=slot, fresh=torch.tensor([True], device=DEV))]
    for t in range(L, L + steps):
        # one token whose three earlier taps come from the conv cache
        m = torch.tensor([[t, t, -t, 0]], dtype=torch.int32, device=DEV)
        q1, k1, v1 = rk.conv_l2(x[t:t + 1], m, w, KD, VD, cache=x)
        assert torch.equal(q1[0], allq[t]) and torch.equal(k1[0], allk[t]) and torch.equal(v1[0], allv[t])
        outs.append(rk.delta_state(heads(q1, 2), heads(k1, 2), heads(v1, 4), gg[t:t + 1], beta[t:t + 1], cu(1), 0.088, state, slots=slot))
    d = dict(q=heads(allq, 2), k=heads(allk, 2), v=heads(allv, 4), g=gg, beta=beta, cu=cu(L + steps), state=state)
    assert_delta(d, 0.088, torch.cat(outs), torch.zeros_like(state), slice(None), slot)
