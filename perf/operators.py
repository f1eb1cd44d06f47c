"""What is measured of the operators that serve one step: the quantised key/value cache (written, read back), attention
over it (each sequence's own pages, and a prefix that all sequences of a batch share), and the gated delta rule with a
carried state.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, 64 where 32 lose what matters)
or, with `own` set, by the framework's entry points.  Layouts are the framework's: q [B, H, M, D] with the query heads
of a key/value head folded into its rows (row r = token r / G), caches [pages, H, page, D], states [slots, HV, value,
key]; a cache row holds e4m3 values and one power of two, stored as a biased exponent byte (255: the row is NaN).
"""
import math
import random

import torch

own = False

LOG2E = 1.4426950408889634
DK = 128  # key and value dimension of a delta-rule head, as in the framework's linear-attention layer


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a batch: each sequence's new token goes to its own page (latency)
        dict(name="write step", op="write", T=64, H=8, D=128, page=16, order="random"),
        # a prefill of four 8192-token prompts, head dim 256: page after page
        dict(name="write prompts", op="write", T=32768, H=8, D=256, page=64, order="pages"),
        # a short history read back so that the prefill attention can go on from it, odd length
        dict(name="read short", op="read", T=1037, H=8, D=128, page=16, order="pages"),
        # a long one, head dim 256
        dict(name="read long", op="read", T=32768, H=8, D=256, page=64, order="pages"),
        # one sequence, one token (latency)
        dict(name="paged one", op="paged", B=1, H=8, G=4, Tq=1, D=128, L=1024, page=16, ragged=False),
        # a batch of ragged histories, two tokens each (one drafted)
        dict(name="paged batch", op="paged", B=64, H=8, G=4, Tq=2, D=128, L=8192, page=16, ragged=True),
        # few long documents, head dim 256
        dict(name="paged long", op="paged", B=8, H=8, G=4, Tq=1, D=256, L=32768, page=64, ragged=False),
        # a chat batch on one system prompt of odd length, short turns
        dict(name="shared chat", op="shared", B=32, H=8, G=4, Tq=1, D=128, Lp=2047, L=512, page=16, ragged=True),
        # many questions on one long document, head dim 256
        dict(name="shared document", op="shared", B=64, H=8, G=4, Tq=1, D=256, Lp=32768, L=1024, page=64, ragged=True),
        # one sequence, one token (latency)
        dict(name="delta one", op="delta", N=1, L=1, H=16, HV=32, ragged=False, fresh=False),
        # a decode step of a batch
        dict(name="delta step", op="delta", N=64, L=1, H=16, HV=32, ragged=False, fresh=False),
        # prompts that start or go on from a state, ragged
        dict(name="delta prompts", op="delta", N=4, L=4096, H=16, HV=32, ragged=True, fresh=True),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["write", "read", "paged", "paged", "shared", "delta", "delta"])
    D = rng.choice([128, 256])
    page = rng.choice([16, 32, 64, 128])
    if op in ("write", "read"):
        H = rng.choice([1, 2, 4, 8])
        return dict(op=op, T=_log(rng, 1, 32768), H=H, D=D, page=page, order=rng.choice(["random", "pages"]))
    if op == "delta":
        H, r = rng.choice([(16, 2), (16, 1), (8, 4), (4, 2), (2, 2)])
        N = _log(rng, 1, 64)
        L = rng.choice([1, 2, _log(rng, 3, 4096)])
        return dict(op=op, N=N if L < 64 else max(1, min(N, 8192 // L)), L=L, H=H, HV=H * r, ragged=rng.random() < 0.5,
                    fresh=rng.random() < 0.5)
    H, G, Tq = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
    if op == "paged":
        B = _log(rng, 1, 64)
        L = min(_log(rng, 16, 65536), (1 << 28) // (B * H * D))
        return dict(op=op, B=B, H=H, G=G, Tq=Tq, D=D, L=max(L, Tq), page=page, ragged=rng.random() < 0.6)
    B = _log(rng, 2, 64)
    Lp = min(_log(rng, 64, 32768), (1 << 34) // (B * H * G * Tq * D))
    return dict(op=op, B=B, H=H, G=G, Tq=Tq, D=D, Lp=Lp, L=max(Tq, _log(rng, 1, 1024)), page=page,
                ragged=rng.random() < 0.6)


def _lengths(n, most, least, ragged):
    """The sequences' lengths: a matter of the case alone.  Ragged ones are spread evenly, the longest among them."""
    if not ragged:
        return [most] * n
    r = random.Random(n * 1000003 + most)
    got = [r.randint(least, most) for _ in range(n)]
    got[r.randrange(n)] = most
    return got


# --------------------------------------------------------------------------------------------------------- quantiser
def _quantise(x):
    """x [..., D] -> e4m3 values [..., D] and biased exponents [...]: the least power of two 2^n with amax <= 448 * 2^n
    (n >= -127), x / 2^n rounded to nearest even.  A row with a value that is not finite is NaN: exponent 255, zeros."""
    x = x.float()
    amax = x.abs().amax(-1)
    fine = torch.isfinite(amax)
    m, e = torch.frexp(torch.where(fine, amax, torch.zeros_like(amax)))  # amax = m * 2^e, m in [0.5, 1)
    n = torch.where(amax > 0, e - 9 + (m > 0.875), torch.full_like(e, -127)).clamp(min=-127)
    y = torch.where(fine[..., None], x, torch.zeros_like(x)) * _pow2(127 - n)[..., None]
    y = y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return y, torch.where(fine, n + 127, torch.full_like(n, 255)).to(torch.uint8)


def _pow2(b):
    """2^(b - 127) for exponent bytes, NaN for 255: by bits, so that it is exact (2^-127 is a subnormal)."""
    b = b.to(torch.int32)
    bits = torch.where(b == 255, torch.full_like(b, 0x7FC00000), torch.where(b == 0, torch.full_like(b, 1 << 22), b << 23))
    return bits.view(torch.float32)


# ---------------------------------------------------------------------------------------------------------- prepare
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(g, n, H, D):
    """Keys or values as a layer makes them: normal, with a spread of magnitudes over rows."""
    return _randn(g, n, H, D) * torch.exp(0.7 * _randn(g, n, H, 1))


def _pool(g, pages, H, page, D):
    """A filled cache.  Quantised in pieces, so that a large one does not need its 32-bit form at once."""
    kc = torch.empty(pages, H, page, D, dtype=torch.float8_e4m3fn, device="cuda")
    vc = torch.empty_like(kc)
    ks = torch.empty(pages, H, page, dtype=torch.uint8, device="cuda")
    vs = torch.empty_like(ks)
    step = max(1, (1 << 26) // (H * page * D))
    for c, s in ((kc, ks), (vc, vs)):
        for a in range(0, pages, step):
            n = min(step, pages - a)
            y, e = _quantise(_rows(g, n * H, page, D).view(n, H, page, D))
            c[a:a + n].view(torch.uint8).copy_(y.view(torch.uint8))
            s[a:a + n] = e
    return dict(kc=kc, ks=ks, vc=vc, vs=vs)


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    op = c["op"]
    if op in ("write", "read"):
        T, H, D, page = c["T"], c["H"], c["D"], c["page"]
        pages = -(-T // page) + 3
        if c["order"] == "random":
            slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].contiguous()
        else:
            at = torch.arange(T, device="cuda")
            slots = torch.randperm(pages, generator=g, device="cuda")[at // page] * page + at % page
        if T > 40:
            slots[7::37] = -1  # the padding of a batch
        if op == "read":
            return dict(op=op, slots=slots, **_pool(g, pages, H, page, D))
        s = _pool(g, pages, H, page, D)
        for t in s.values():
            t.view(torch.uint8).zero_()
        k = _rows(g, T, H, D).bfloat16()
        return dict(op=op, slots=slots, k=k, v=_rows(g, T, H, D).bfloat16(), **s)
    if op in ("paged", "shared"):
        B, H, D, page, M = c["B"], c["H"], c["D"], c["page"], c["Tq"] * c["G"]
        Lp = c.get("Lp", 0)
        lens = _lengths(B, c["L"], c["Tq"], c["ragged"])
        P, PP = -(-c["L"] // page), -(-Lp // page)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + PP + 1
        s = _pool(g, pages, H, page, D)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.zeros(B, P, dtype=torch.int32, device="cuda")
        at = PP
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        # the new tokens are the last ones of each history; positions count from the prefix's start
        last = torch.tensor(lens, dtype=torch.int32).cuda()[:, None] + Lp
        qpos = (last - c["Tq"] + torch.arange(c["Tq"], dtype=torch.int32, device="cuda")).contiguous()
        q = (_randn(g, B, H, M, D) * 0.5).bfloat16()
        return dict(op=op, q=q, table=table, qpos=qpos, G=c["G"], scale=D ** -0.5, prefix=order[:PP].contiguous() if Lp else None,
                    Lp=Lp, **s)
    N, H, HV = c["N"], c["H"], c["HV"]
    lens = _lengths(N, c["L"], 1, c["ragged"])
    T = sum(lens)
    cu = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).cuda()
    silu = torch.nn.functional.silu  # what the layer's convolution leaves
    unit = lambda x: (x / x.square().sum(-1, keepdim=True).sqrt()).bfloat16()  # noqa: E731
    S = N + 2
    return dict(op=op, q=unit(silu(_randn(g, T, H, DK))), k=unit(silu(_randn(g, T, H, DK))), v=silu(_randn(g, T, HV, DK)).bfloat16(),
                beta=torch.sigmoid(_randn(g, T, HV)).bfloat16(), g=-torch.nn.functional.softplus(_randn(g, T, HV) - 2.0) * LOG2E,
                cu=cu, scale=DK ** -0.5, state=_randn(g, S, HV, DK, DK) * 0.2, L=c["L"],
                slots=torch.randperm(S, generator=g, device="cuda")[:N].to(torch.int32),
                fresh=(torch.arange(N, device="cuda") % 2 == 0) if c["fresh"] else None)


# -------------------------------------------------------------------------------------------------------------- run
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from reax_engine_kernels_b200 import kernels as rk

    op = s["op"]
    if op == "delta":
        o = rk.delta_state(s["q"], s["k"], s["v"], s["g"], s["beta"], s["cu"], s["scale"], s["state"], slots=s["slots"], fresh=s["fresh"])
        return dict(o=o, state=s["state"])
    cache = rk.KvCache(s["kc"], s["ks"], s["vc"], s["vs"])
    if op == "write":
        rk.kv_write(s["k"], s["v"], cache, s["slots"])
        return dict(kc=s["kc"], ks=s["ks"], vc=s["vc"], vs=s["vs"])
    if op == "read":
        return rk.kv_read(cache, s["slots"])
    if op == "shared":
        return rk.fmha_paged(s["q"], cache, s["table"], s["scale"], qpos=s["qpos"], G=s["G"], prefix=s["prefix"], prefix_len=s["Lp"])
    return rk.fmha_paged(s["q"], cache, s["table"], s["scale"], qpos=s["qpos"], G=s["G"])


def _run_plain(s):
    op = s["op"]
    if op == "write":
        page = s["kc"].shape[2]
        at = (s["slots"] >= 0).nonzero()[:, 0]
        pg, off = s["slots"][at] // page, s["slots"][at] % page
        for x, c, e in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
            y, n = _quantise(x[at])
            c.view(torch.uint8)[pg, :, off] = y.view(torch.uint8)
            e[pg, :, off] = n
        return dict(kc=s["kc"], ks=s["ks"], vc=s["vc"], vs=s["vs"])
    if op == "read":
        return tuple(_read_plain(c, e, s["slots"]) for c, e in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
    if op in ("paged", "shared"):
        return _attention_plain(s)
    return _delta_plain(s)


def _read_plain(c, e, slots):
    page = c.shape[2]
    at = slots.clamp(min=0)
    pg, off = at // page, at % page
    x = c.view(torch.uint8)[pg, :, off].view(torch.float8_e4m3fn).float() * _pow2(e[pg, :, off])[..., None]
    return torch.where((slots >= 0)[:, None, None], x, torch.zeros_like(x)).bfloat16()


def _gather(c, e, table):
    """The pages of a table [..., P] as 32-bit rows [..., H, P * page, D]."""
    x = c.view(torch.uint8)[table.long()].view(torch.float8_e4m3fn).float() * _pow2(e[table.long()])[..., None]
    x = x.movedim(-3, -4)
    return x.reshape(*x.shape[:-3], x.shape[-3] * x.shape[-2], x.shape[-1])


def _attention_plain(s):
    q, Lp = s["q"].float(), s["Lp"]
    B, H, M, D = q.shape
    last = s["qpos"].repeat_interleave(s["G"], 1)[:, None, :, None]  # [B, 1, M, 1]
    k, v = _gather(s["kc"], s["ks"], s["table"]), _gather(s["vc"], s["vs"], s["table"])
    n = k.shape[2]
    x = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    pos = Lp + torch.arange(n, device=q.device)
    x = torch.where(pos <= last, x, torch.full_like(x, -math.inf))
    if s["prefix"] is not None:
        kp, vp = _gather(s["kc"], s["ks"], s["prefix"]), _gather(s["vc"], s["vs"], s["prefix"])  # [H, n, D]
        rows = q.transpose(0, 1).reshape(H, B * M, D)
        xp = (torch.matmul(rows, kp.transpose(-1, -2)) * s["scale"]).view(H, B, M, -1).transpose(0, 1)
        pos = torch.arange(kp.shape[1], device=q.device)
        xp = torch.where((pos < Lp) & (pos <= last), xp, torch.full_like(xp, -math.inf))
        x = torch.cat([xp, x], -1)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    norm = p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., p.shape[-1] - n:], v)
    if s["prefix"] is not None:
        pp = p[..., :p.shape[-1] - n].transpose(0, 1).reshape(H, B * M, -1)
        o = o + torch.matmul(pp, vp).view(H, B, M, D).transpose(0, 1)
    return torch.where(norm > 0, o / norm, torch.zeros_like(o)).bfloat16()


def _delta_plain(s):
    """Chunks of up to 64 tokens: within a chunk the updates are solved together, from chunk to chunk the state goes on."""
    cu, L, state = s["cu"], s["L"], s["state"]
    N, T, HV = cu.shape[0] - 1, s["q"].shape[0], s["v"].shape[1]
    rep = HV // s["q"].shape[1]
    C = min(64, 1 << (L - 1).bit_length())
    n = -(-L // C)
    at = cu[:-1, None] + torch.arange(n * C, device=cu.device)
    live = at < cu[1:, None]
    at = at.clamp(max=T - 1)

    def chunks(x):  # [T, heads, ...] -> [N, heads, n, C, ...], zeros past a sequence's end
        x = torch.where(live.view(N, n * C, *[1] * (x.dim() - 1)), x[at].float(), 0.0)
        return x.transpose(1, 2).reshape(N, x.shape[2], n, C, *x.shape[3:])

    q, k = (chunks(s[w]).repeat_interleave(rep, 1) for w in ("q", "k"))
    v, beta, g = chunks(s["v"]), chunks(s["beta"]), chunks(s["g"]).double().cumsum(-1)
    lower = torch.ones(C, C, device=cu.device).tril()
    decay = (torch.exp2((g[..., :, None] - g[..., None, :]) * lower) * lower).float()
    strict = (beta[..., None] * decay * torch.matmul(k, k.transpose(-1, -2))).double().tril(-1)
    solve = torch.eye(C, device=cu.device, dtype=torch.float64) - strict  # (1 + strict)^-1 by doubling: strict^C = 0
    power = strict
    for _ in range(max(0, C.bit_length() - 2)):
        power = power @ power
        solve = solve + solve @ power
    solve = solve.float()
    grow = torch.exp2(g).float()
    u = solve @ (beta[..., None] * v)
    w = solve @ ((beta * grow)[..., None] * k)
    inner = torch.matmul(q, k.transpose(-1, -2)) * decay
    left = torch.exp2(g[..., -1:] - g).float()
    slots = s["slots"].long()
    h = state[slots]
    if s["fresh"] is not None:
        h = torch.where(s["fresh"][:, None, None, None], 0.0, h)
    o = torch.empty(N, HV, n, C, DK, device=cu.device)
    for i in range(n):
        ht = h.transpose(-1, -2)
        new = u[:, :, i] - w[:, :, i] @ ht
        o[:, :, i] = (q[:, :, i] * grow[:, :, i, :, None]) @ ht + inner[:, :, i] @ new
        h = h * grow[:, :, i, -1:, None] + (new * left[:, :, i, :, None]).transpose(-1, -2) @ k[:, :, i]
    state[slots] = h
    out = (o * s["scale"]).reshape(N, HV, n * C, DK).transpose(1, 2)[live]
    return dict(o=out.bfloat16(), state=state)


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    op = c["op"]
    if op in ("write", "read"):
        n = c["T"] - (len(range(7, c["T"], 37)) if c["T"] > 40 else 0)
        rows = 2 * n * c["H"]
        wide = 2 * c["D"] * (rows if op == "write" else 2 * c["T"] * c["H"])
        return dict(bytes=wide + rows * (c["D"] + 1) + 8 * c["T"], flops=2 * rows * c["D"])
    if op in ("paged", "shared"):
        M, Lp, D = c["Tq"] * c["G"], c.get("Lp", 0), c["D"]
        lens = _lengths(c["B"], c["L"], c["Tq"], c["ragged"])
        seen = sum(lens) + Lp
        pages = sum(-(-n // c["page"]) for n in lens) + -(-Lp // c["page"])
        pairs = c["G"] * sum(n - c["Tq"] + 1 + t + Lp for n in lens for t in range(c["Tq"]))
        return dict(bytes=2 * seen * c["H"] * (D + 1) + 4 * c["B"] * c["H"] * M * D + 4 * pages + 4 * c["B"] * c["Tq"],
                    flops=4 * D * c["H"] * pairs)
    lens = _lengths(c["N"], c["L"], 1, c["ragged"])
    T, N = sum(lens), c["N"]
    read = N - (N + 1) // 2 if c["fresh"] else N
    return dict(bytes=(read + N) * c["HV"] * DK * DK * 4 + T * (2 * c["H"] * DK * 2 + 2 * c["HV"] * DK * 2 + c["HV"] * 6) + 12 * N,
                flops=7 * DK * DK * c["HV"] * T)


# ------------------------------------------------------------------------------------------------------------ exact
def _e4m3_table():
    """The 256 values of e4m3 from its definition: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f and 0xff NaN."""
    got = []
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        x = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        got.append(math.nan if b & 127 == 127 else -x if b & 128 else x)
    return torch.tensor(got, dtype=torch.float64, device="cuda")


def _exact_rows(c, e):
    p = torch.pow(2.0, e.double() - 127.0)
    return _e4m3_table()[c.view(torch.uint8).long()] * torch.where(e == 255, math.nan, p)[..., None]


def _exact_write(x, slots, shape):
    """x / 2^n as numbers (not rounded to e4m3), at their places."""
    pages, H, page, D = shape
    out = torch.zeros(pages * page, H, D, dtype=torch.float64, device="cuda")
    for a in range(0, x.shape[0], 2048):  # in pieces, to bound the memory
        y, at = x[a:a + 2048].double(), slots[a:a + 2048]
        big = y.abs().amax(-1, keepdim=True)
        n = torch.ceil(torch.log2(torch.where(big > 0, big, 1.0) / 448.0))
        n = torch.where(448.0 * 2.0 ** n < big, n + 1, torch.where(448.0 * 2.0 ** (n - 1) >= big, n - 1, n)).clamp(min=-127)
        out[at[at >= 0]] = (y / 2.0 ** n)[at >= 0]
    return out.view(pages, page, H, D).transpose(1, 2).contiguous()


def _exact_attention(s):
    q, Lp, G = s["q"].double(), s["Lp"], s["G"]
    B, H, M, D = q.shape
    page, out = s["kc"].shape[2], torch.zeros_like(q)
    ends = s["qpos"].tolist()
    for b in range(B):
        n = max(ends[b]) + 1 - Lp
        own_pages = s["table"][b, :-(-n // page)].long()
        parts = [(own_pages, n)] if s["prefix"] is None else [(s["prefix"].long(), Lp), (own_pages, n)]
        for h in range(H):
            k, v = (torch.cat([_exact_rows(c[pg, h], e[pg, h]).reshape(-1, D)[:m] for pg, m in parts])
                    for c, e in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
            for r in range(M):
                m = ends[b][r // G] + 1
                p = torch.softmax((k[:m] @ q[b, h, r]) * s["scale"], 0)
                out[b, h, r] = p @ v[:m]
    return out


def _exact_delta(s):
    cu, state = s["cu"].tolist(), s["state"].double()
    q, k, v, beta, g = (s[w].double() for w in ("q", "k", "v", "beta", "g"))
    rep = v.shape[1] // q.shape[1]
    o = torch.zeros_like(v)
    lens = [b - a for a, b in zip(cu, cu[1:])]
    slots = s["slots"].tolist()
    h = torch.stack([state[i] for i in slots])
    if s["fresh"] is not None:
        h[s["fresh"]] = 0.0
    starts = torch.tensor(cu[:-1], device="cuda")
    for t in range(max(lens)):  # token by token, the sequences that still have one together
        on = torch.tensor([i for i, n in enumerate(lens) if n > t], device="cuda")
        at = starts[on] + t
        kt, qt = (x[at].repeat_interleave(rep, 1)[..., None] for x in (k, q))
        x = h[on] * torch.pow(2.0, g[at])[..., None, None]
        d = beta[at][..., None] * (v[at] - (x @ kt)[..., 0])
        x = x + d[..., None] * kt.transpose(-1, -2)
        h[on] = x
        o[at] = s["scale"] * (x @ qt)[..., 0]
    for i, j in enumerate(slots):
        state[j] = h[i]
    return dict(o=o, state=state)


def exact(case, seed):
    op = case["op"]
    if op in ("paged", "shared"):
        lens = _lengths(case["B"], case["L"], case["Tq"], case["ragged"])
        if case["B"] * case["H"] * case["G"] * case["Tq"] * 1.5e-4 + (sum(lens) + case.get("Lp", 0) * case["B"]) * case["H"] * case["D"] * 2e-9 > 15:
            return None
    s = prepare(case, seed)
    if op == "write":
        shape = s["kc"].shape
        return dict(kc=_exact_write(s["k"], s["slots"], shape), ks=None, vc=_exact_write(s["v"], s["slots"], shape), vs=None)
    if op == "read":
        page, at = s["kc"].shape[2], s["slots"].clamp(min=0)
        got = [_exact_rows(c.view(torch.uint8)[at // page, :, at % page],
                           e[at // page, :, at % page]) for c, e in ((s["kc"], s["ks"]), (s["vc"], s["vs"]))]
        return tuple(torch.where((s["slots"] >= 0)[:, None, None], x, 0.0) for x in got)
    if op in ("paged", "shared"):
        for w in ("kc", "vc"):
            s[w] = s[w].view(torch.uint8)
        return _exact_attention(s)
    return _exact_delta(s)
