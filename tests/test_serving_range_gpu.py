"""Attention over the quantised cache where keys and values of very different powers of two meet, on the GPU against the
formula in 64 bits.  What a key adds is bounded by its own weight here: no term of the tolerance takes the largest value alone.

Tolerance of a row, with p_j the weights, n their number, v_j = row of e4m3 values * 2^nv_j:
  * each weight is rounded to f16 (2^-11 of it), its exponent is off by the score's error (a dot product of D terms and its scaling
    in fp32: (D + 8) * 2^-24 of the sum of its terms' magnitudes) and by 2^-24 of a difference of at most 150 in the log2 domain, twice,
    with ex2's own 2^-22 (2^-16 in all), and the sum of n terms in fp32 by n * 2^-24 of their magnitudes;
  * the divisor is off by the same without the f16 rounding;
  * below f16's normal range a weight is off by 2^-25 against a largest p_j 2^nv_j of at least one, and e4m3 values reach 448:
    n * 2^-25 * 448 * max_j p_j 2^nv_j;
  * weights under 2^-126 of the row's largest are zero, and the products p_j 2^nv_j are held to 2^-150: n * 448 * 2^-150;
  * the result is rounded to bf16, 2^-8 of it, 2^-134 below bf16's normal range."""
import math
import random

import pytest
import torch

from reax_engine_kernels_b200 import kernels as rk
from tests.test_serving_gpu import BF, DEV, gen, randn, status, value_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clear_status():
    status()
    yield
    assert status() == 0, "a kernel reported something that the test did not expect"


def assert_rows(o, q, c, table, scale, qpos, G, prefix=None, Lp=0, rows=None):
    """Rows (b, r) of all heads (all of them by default) against the formula in 64 bits, within the tolerance above.  Keys of pages
    that are not there are not seen; a NaN row among those that are makes the result NaN."""
    B, H, M, D = q.shape
    page = c.k.shape[2]
    kc, vc = (t.view(torch.uint8) for t in (c.k, c.v))
    pages = torch.zeros(0, dtype=torch.int64, device=DEV) if prefix is None else prefix.long()
    for b, r in rows if rows is not None else [(b, r) for b in range(B) for r in range(M)]:
        n = min(int(qpos[b, r // G]) + 1, Lp + table.shape[1] * page)
        j = torch.arange(max(n, 0), device=DEV)
        pg, off = torch.empty_like(j), torch.where(j < Lp, j, j - Lp) % page
        pg[j < Lp] = pages[j[j < Lp] // page]
        pg[j >= Lp] = table[b].long()[(j[j >= Lp] - Lp) // page]
        there = (pg >= 0) & (pg < c.k.shape[0])
        pg, off, n = pg[there], off[there], int(there.sum())
        if n == 0:
            assert o[b, :, r].count_nonzero() == 0, (b, r)
            continue
        k, v = (value_ref(t[pg, :, off], e[pg, :, off]) for t, e in ((kc, c.ke), (vc, c.ve)))  # [n, H, D]
        nan = (torch.isnan(k) | torch.isnan(v)).any(-1).any(0)  # [H]
        nv = torch.pow(2.0, c.ve[pg, :, off].double() - 127).T  # [H, n]
        qr = q[b, :, r].double()
        p = torch.softmax(torch.einsum("hd,nhd->hn", qr, k) * scale, -1)
        off_by = (D + 8) * 2.0 ** -24 * torch.einsum("hd,nhd->hn", qr.abs(), k.abs()) * abs(scale) + 2.0 ** -16 + n * 2.0 ** -24
        want = torch.einsum("hn,nhd->hd", p, v)
        tol = torch.einsum("hn,nhd->hd", p * (off_by + 2.0 ** -11), v.abs()) + (p * off_by).sum(-1)[:, None] * want.abs()
        tol = tol * 1.01 + (n * 2.0 ** -25 * 448 * (p * nv).amax(-1) + n * 2.0 ** -126 * v.abs().amax((0, 2)))[:, None] + 2.0 ** -8 * want.abs()
        tol = tol + n * 448 * 2.0 ** -150 + 2.0 ** -134
        got = o[b, :, r].double()
        assert torch.isfinite(got[~nan]).all() and torch.isnan(got[nan]).all(), (b, r)
        worst = ((got - want).abs() - tol)[~nan]
        assert worst.numel() == 0 or worst.max() <= 0, (b, r, worst.max().item())


def cached(g, lens, H, page, D, Lp):
    """A cache with the pages of `lens` and of a prefix, unwritten; and what addresses it: table, prefix, the slots of the
    prefix and of each sequence."""
    PP = -(-Lp // page)
    need = [-(-n // page) for n in lens]
    c = rk.kv_cache(sum(need) + PP + 1, H, page, D)
    order = torch.randperm(c.k.shape[0], generator=g, device=DEV)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV)
    at, slots = PP, []
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(torch.int32)
        j = torch.arange(lens[b], device=DEV)
        slots.append(order[at + j // page] * page + j % page)
        at += n
    j = torch.arange(Lp, device=DEV)
    return c, table, order[:PP].to(torch.int32).contiguous(), order[j // page] * page + j % page, slots


def along(g, B, H, M, D):
    """A direction per head, and query rows that are multiples of it: with a scale of ln 2 / D a key t * direction has the score
    t, 1.5 t or 2 t in the log2 domain."""
    w = torch.where(randn(g, H, D) < 0, -1.0, 1.0)
    f = torch.tensor([1.0, 1.5, 2.0, 1.0], device=DEV)[torch.arange(M, device=DEV) % 4]
    return w, (w[:, None, :] * f[:, None]).expand(B, H, M, D).to(BF).contiguous()


# rows of 8 and of 16 leave no padding row in a tile, which would raise the references for its neighbours
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("gap", [60, 104, 124, 130, 208])
@pytest.mark.parametrize("M,Lp,L", [(8, 0, 13), (8, 0, 200), (8, 0, 3000), (16, 0, 200), (3, 0, 200), (4, 330, 20), (16, 330, 20)])
def test_zero_value_row_under_the_largest_weight(M, Lp, L, gap, D):
    """A key far above all others whose value row is zero, before values of 512 and more: what is left of the others' weights counts."""
    g = gen(gap + D)
    B, H, page = 4 if M == 4 else 1, 2, 16
    c, table, prefix, pslots, slots = cached(g, [L] * B, H, page, D, Lp)
    w, q = along(g, B, H, M, D)
    for s in ([pslots] if Lp else []) + slots:
        k, v = randn(g, len(s), H, D) * 0.3, randn(g, len(s), H, D) * 1000
        for at in (0, 70):  # in the first group of 16 keys, and behind others
            if at < len(s):
                k[at], v[at] = w * float(gap), 0.0
        rk.kv_write(k.to(BF), v.to(BF), c, s)
    qpos = torch.full((B, M), Lp + L - 1, dtype=torch.int32, device=DEV)
    scale = math.log(2) / D
    o = rk.fmha_paged(q, c, table, scale, qpos=qpos, prefix=prefix if Lp else None, prefix_len=Lp)
    assert_rows(o, q, c, table, scale, qpos, 1, prefix if Lp else None, Lp)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("M,Lp,L", [(8, 0, 200), (16, 0, 200), (8, 0, 3000), (16, 330, 20), (64, 330, 20)])
def test_smallest_values(M, Lp, L, D):
    """Values whose power of two is the least there is, 2^-127 (a row in some hundred 2^-126), and results below fp32's normal range."""
    g = gen(M + D)
    H, page = 2, 16
    c, table, prefix, pslots, slots = cached(g, [L], H, page, D, Lp)
    for s in ([pslots] if Lp else []) + slots:
        rk.kv_write(randn(g, len(s), H, D).to(BF), (randn(g, len(s), H, D) * 6e-37).to(BF), c, s)
    assert c.ve.min() == 0 and c.ve.max() <= 1
    q = randn(g, 1, H, M, D).to(BF)
    qpos = torch.full((1, M), Lp + L - 1, dtype=torch.int32, device=DEV)
    o = rk.fmha_paged(q, c, table, 0.1, qpos=qpos, prefix=prefix if Lp else None, prefix_len=Lp)
    assert o.count_nonzero() > o.numel() * 0.9
    assert_rows(o, q, c, table, 0.1, qpos, 1, prefix if Lp else None, Lp)


# M = 16 rows of one sequence keep the prefix with the kernel for few rows, 64 take it to the one of 128-row tiles, whose tiles have
# 64 keys; 8 and 16 rows without a prefix
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("M,H,Lp,L", [(8, 2, 0, 400), (16, 2, 0, 400), (16, 2, 400, 20), (64, 2, 400, 20), (64, 16, 2400, 20)])
@pytest.mark.parametrize("kind", ["zero on top", "large value", "huge value", "tile of large values", "large key", "small values", "masked"])
def test_rows_that_weigh_nothing_take_nothing_from_the_others(kind, M, H, Lp, L, D):
    """Rows of another magnitude whose weight is next to nothing, or which some queries do not see: the result is the others', as
    exactly as without them."""
    g = gen(M + H + D)
    page = 16
    c, table, prefix, pslots, slots = cached(g, [L], H, page, D, Lp)
    w, q = along(g, 1, H, M, D)
    where, n = (pslots, Lp) if Lp else (slots[0], L)
    if Lp:
        rk.kv_write((randn(g, L, H, D) * 0.3 - w).to(BF), randn(g, L, H, D).to(BF), c, slots[0])
    k, v = randn(g, n, H, D) * 0.3, randn(g, n, H, D)
    qpos = torch.full((1, M), Lp + L - 1, dtype=torch.int32, device=DEV)
    at = torch.arange(5, n, 64, device=DEV)  # one in each tile of 64 keys
    if kind == "zero on top":
        k[at], v[at] = w * 104.0, 0.0
    elif kind == "large value":
        k[at], v[at] = -60.0 * w, v[at] * 2.0 ** 30
    elif kind == "huge value":
        k[at], v[at] = -104.0 * w, v[at] * 2.0 ** 80
    elif kind == "tile of large values":
        k[64:128], v[64:128] = -60.0 * w, v[64:128] * 2.0 ** 40
        k[256:320], v[256:320] = -104.0 * w, v[256:320] * 2.0 ** 70
    elif kind == "large key":
        k[at] = -w * 2.0 ** 30
    elif kind == "small values":  # almost all the weight on rows 2^-30 of their neighbours
        k[at], v[at] = 104.0 * w, v[at] * 2.0 ** -30
        k[at + 1], v[at + 1] = 80.0 * w, v[at + 1] * 2.0 ** -20
    else:  # the last rows of the keys, which half of the queries do not see
        k[n - 20:], v[n - 20:] = k[n - 20:] * 2.0 ** 20, v[n - 20:] * 2.0 ** 100
        qpos[:, :M // 2] = n - 21
    rk.kv_write(k.to(BF), v.to(BF), c, where)
    scale = math.log(2) / D
    if kind == "masked":
        q[:, :, M // 2:] *= 2.0 ** -24  # scores of fp32's range where the large keys are seen
    o = rk.fmha_paged(q, c, table, scale, qpos=qpos, prefix=prefix if Lp else None, prefix_len=Lp)
    assert_rows(o, q, c, table, scale, qpos, 1, prefix if Lp else None, Lp, rows=[(0, r) for r in range(0, M, max(1, M // 12))])


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("M", [8, 64])
def test_rows_that_see_nothing_of_far_magnitudes(M, D):
    """The least qpos there is, and others below the prefix or inside it, over tiles of the prefix with rows far apart."""
    g = gen(M + D)
    H, page, Lp, L, B = 2, 16, 400, 20, 2
    c, table, prefix, pslots, slots = cached(g, [L] * B, H, page, D, Lp)
    for s in [pslots] + slots:
        v = randn(g, len(s), H, D) * torch.exp2(10.0 * randn(g, len(s), H, 1))
        rk.kv_write(randn(g, len(s), H, D).to(BF), v.to(BF), c, s)
    qpos = torch.full((B, M), Lp + L - 1, dtype=torch.int32, device=DEV)
    qpos[0, :6] = torch.tensor([-(1 << 31), -(1 << 31) + 1, -2, -1, 0, 64], dtype=torch.int32)
    q = randn(g, B, H, M, D).to(BF)
    o = rk.fmha_paged(q, c, table, D ** -0.5, qpos=qpos, prefix=prefix, prefix_len=Lp)
    assert o[0, :, :4].count_nonzero() == 0
    assert_rows(o, q, c, table, D ** -0.5, qpos, 1, prefix, Lp, rows=[(0, r) for r in range(8)] + [(1, 0)])


@pytest.mark.parametrize("seed", range(12))
def test_far_magnitudes_drawn(seed):
    """Rows of all magnitudes and zero rows, with queries that see part of them, prefixes that end inside a tile, pages that are
    not there and NaN rows: everything that a tile may hold, together.  The same bits on a second run."""
    r, g = random.Random(seed), gen(seed)
    H, D, page, Lp = r.choice([1, 2, 5]), r.choice([128, 256]), r.choice([16, 48, 64]), [0, 130, 700, 1601][seed % 4]
    B, G, Tq = r.choice([(1, 8, 1), (2, 8, 2), (3, 4, 3), (9, 8, 1), (20, 5, 2)])
    lens = [r.randint(Tq, 300) for _ in range(B)]
    c, table, prefix, pslots, slots = cached(g, lens, H, page, D, Lp)
    for s in ([pslots] if Lp else []) + slots:
        n = len(s)
        k = randn(g, n, H, D) * torch.exp2((r.choice([0.3, 5.0]) * randn(g, n, H, 1)).clamp(-60, 18))
        v = randn(g, n, H, D) * torch.exp2((r.choice([2.0, 15.0]) * randn(g, n, H, 1)).clamp(-110, 100))
        v[torch.rand(n, H, generator=g, device=DEV) < 0.03] = 0
        k[torch.rand(n, H, generator=g, device=DEV) < 0.001] = math.nan
        rk.kv_write(k.to(BF), v.to(BF), c, s)
    missing = Lp > page and seed % 3 == 0
    if missing:
        prefix[1] = c.k.shape[0]
    qpos = torch.tensor([sorted(r.randint(-1, Lp + n - 1) for _ in range(Tq - 1)) + [Lp + n - 1] for n in lens], dtype=torch.int32, device=DEV)
    q = (randn(g, B, H, G * Tq, D) * r.choice([0.3, 3.0])).to(BF)
    kw = dict(qpos=qpos, G=G, prefix=prefix if Lp else None, prefix_len=Lp)
    o, o2 = (rk.fmha_paged(q, c, table, D ** -0.5, **kw) for _ in range(2))
    assert status() == (0x502 if missing else 0)
    assert torch.equal(o.view(torch.int16), o2.view(torch.int16))
    assert_rows(o, q, c, table, D ** -0.5, qpos, G, kw["prefix"], Lp)
