"""Launches of the serving entry points that only large batches reach, on the GPU against the formulas in 64 bits: the join
of many rows, the longer chunks of a full GPU, more than 256 sequences of the delta rule, refused slots among long sequences; and
the accuracy of the delta rule's state."""
import math

import pytest
import torch

from reax_engine_kernels_b200 import kernels as rk
from tests.test_serving_gpu import BF, DEV, assert_delta, delta_inputs, delta_ref, gen, setup, status
from tests.test_serving_range_gpu import assert_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clear_status():
    status()
    yield
    assert status() == 0, "a kernel reported something that the test did not expect"


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("G,Tq,most,Lp", [(4, 2, 3000, 0), (8, 2, 2100, 0), (4, 2, 1000, 700)])
def test_batch_that_fills_the_gpu(G, Tq, most, Lp, D):
    """64 sequences of 8 heads: 512 tiles of rows and more, 4096 rows and more to join, several chunks each."""
    B, H = 64, 8
    assert B * H * G * Tq > 8 * torch.cuda.get_device_properties(0).multi_processor_count
    lens = [Tq + (b * b * 37) % (most - Tq) for b in range(B)]
    lens[5], lens[6], lens[63] = most, Tq, 1024
    q, c, table, qpos, prefix = setup(D + G, B, H, G, Tq, D, 16, lens, Lp)
    kw = dict(qpos=qpos, G=G, prefix=prefix if Lp else None, prefix_len=Lp)
    o = rk.fmha_paged(q, c, table, D ** -0.5, **kw)
    M = G * Tq
    rows = [(b, (b * 7 + i) % M) for b in (0, 5, 6, 17, 40, 63) for i in (0, G)]
    assert_rows(o, q, c, table, D ** -0.5, qpos, G, kw["prefix"], Lp, rows=rows)
    # all the others agree with a batch of eight, whose launch is another, in the 2-norm of a row: two roundings to bf16, and two of
    # each weight to f16, which do not know the values' signs and so add up as the values themselves do
    for a in range(0, B, 8):
        s = slice(a, a + 8)
        part = rk.fmha_paged(q[s], c, table[s], D ** -0.5, **{**kw, "qpos": qpos[s]}).double()
        assert ((o[s].double() - part).norm(dim=-1) <= (2 * 2.0 ** -8 + 2 * 2.0 ** -11) * part.norm(dim=-1)).all()


def test_delta_state_many_sequences():
    """More than 256 sequences, which are not put in order of their length: most of one token, some of none, some for either kernel."""
    lens = [1] * 300
    for i, n in ((0, 15), (3, 0), (100, 14), (255, 33), (256, 64), (270, 2), (299, 40)):
        lens[i] = n
    d = delta_inputs(41, lens, 1, 2, 301, behind=3)
    slots = torch.randperm(301, generator=gen(1), device=DEV)[:300].to(torch.int32)
    slots[7] = -1
    state0, T = d["state"].clone(), d["q"].shape[0]
    o = torch.full((T, 2, 128), 7.0, dtype=BF, device=DEV)
    rk.delta_state(*(d[n] for n in ("q", "k", "v", "g", "beta", "cu")), 0.1, d["state"], slots=slots, o=o)
    left = int(d["cu"][7])
    assert (o[sum(lens):] == 7).all() and (o[left] == 7).all()
    live = torch.tensor([t for t in range(sum(lens)) if t != left], device=DEV)
    assert_delta(d, 0.1, o, state0, live, slots)


def test_delta_state_slots_of_long_sequences():
    """Sequences of both kernels: a slot past the end, one named before by a sequence of the other kernel or of the same, a negative one,
    one that only an empty sequence has named."""
    #        ok   past  dup of 0  left  ok  dup of 4  ok  empty  ok (7 has no tokens)  dup of 6, short
    lens = [20, 40, 3, 33, 64, 17, 2, 0, 50, 30, 5]
    slots = torch.tensor([1, 9, 1, -4, 4, 4, 0, 7, 7, 0, 1 << 30], dtype=torch.int32, device=DEV)
    d = delta_inputs(42, lens, 2, 4, 9)
    state0, cu = d["state"].clone(), d["cu"].tolist()
    o = torch.full((sum(lens), 4, 128), 7.0, dtype=BF, device=DEV)
    rk.delta_state(*(d[n] for n in ("q", "k", "v", "g", "beta", "cu")), 0.1, d["state"], slots=slots, o=o)
    assert status() == 0x503
    runs = (0, 4, 6, 8)
    for i in range(len(lens)):
        part = o[cu[i]:cu[i + 1]]
        assert torch.isfinite(part).all() if i in runs else (part == 7).all() if i == 3 else torch.isnan(part).all()
    ref = torch.tensor([int(s) if i in runs else -1 for i, s in enumerate(slots)], dtype=torch.int32, device=DEV)
    live = torch.cat([torch.arange(cu[i], cu[i + 1], device=DEV) for i in runs])
    assert_delta(d, 0.1, o, state0, live, ref)


def _cut(x):
    """The 16 leading bits of a number: the sum of two bf16 terms."""
    a = x.to(BF).double()
    return a + (x - a).to(BF).double()


def test_delta_state_holds_24_bits():
    """The state of a prompt in its 2-norm.  Between two forgettings a chunk's state takes about 71 roundings to fp32 of half a step or
    less (24 + 40 of the accumulations in h k and T r that make up u, 6 of the update's and one of the decay), each independent of
    the others: sqrt(71) * 2^-24 of the norm.  (The bound per row that the other tests use grows with the number of tokens and would let
    16 bits pass.)  The recurrence with h and u cut to 16 bits is far outside."""
    limit = math.sqrt(71) * 2.0 ** -24
    for lens in ([320, 500, 47], [1000]):
        d = delta_inputs(43 + len(lens), lens, 2, 4, len(lens))
        state0 = d["state"].clone()
        rk.delta_state(*(d[n] for n in ("q", "k", "v", "g", "beta", "cu")), 0.1, d["state"])
        ref = delta_ref({**d, "state": state0}, 0.1)[2]
        for n in range(len(lens)):
            assert (d["state"][n].double() - ref[n]).norm() <= limit * ref[n].norm(), n
    h, cu = state0[0].double(), d["cu"].tolist()
    rep = 2
    for t in range(cu[0], cu[1]):
        kt = d["k"][t].double().repeat_interleave(rep, 0)[..., None]
        h = _cut(h * torch.exp2(d["g"][t].double())[:, None, None])
        u = _cut(d["beta"][t].double()[:, None] * (d["v"][t].double() - (h @ kt)[..., 0]))
        h = h + u[..., None] * kt.transpose(-1, -2)
    assert (h - ref[0]).norm() > 2 * limit * ref[0].norm()
