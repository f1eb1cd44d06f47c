"""Refusals of the serving entry points (quantised cache, paged attention, delta rule with a state), without a GPU: the
front end checks types and shapes before it touches a device, the C entry points check theirs before they launch."""
import ctypes

import pytest
import torch

from reax_engine_kernels_b200 import abi
from reax_engine_kernels_b200 import kernels as rk

BF = torch.bfloat16


def cache(pages=3, H=2, page=16, D=128):
    return rk.kv_cache(pages, H, page, D, device="cpu")


def kv(T=4, H=2, D=128, dtype=BF):
    return torch.zeros(T, H, D, dtype=dtype), torch.zeros(T, H, D, dtype=dtype), torch.zeros(T, dtype=torch.int64)


def test_cache_layout():
    c = cache(5, 3, 32, 256)
    assert c.k.shape == c.v.shape == (5, 3, 32, 256) and c.k.dtype == torch.float8_e4m3fn
    assert c.ke.shape == c.ve.shape == (5, 3, 32) and c.ke.dtype == torch.uint8


@pytest.mark.parametrize("change, words", [
    (dict(D=64), "head dimension"),
    (dict(dtype=torch.float16), "bfloat16"),
    (dict(slots=torch.zeros(4, dtype=torch.int32)), "int64"),
    (dict(slots=torch.zeros(5, dtype=torch.int64)), "shape"),
    (dict(cache=lambda: cache(H=3)), "cache.k"),
    (dict(cache=lambda: cache(D=256)), "cache.k"),
    (dict(cache=lambda: cache(page=24)), "multiple of 16"),
    (dict(cache=lambda: cache()._replace(ke=torch.zeros(3, 2, 16, dtype=torch.int8))), "uint8"),
    (dict(cache=lambda: cache()._replace(v=torch.zeros(6, 2, 16, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)[::2])), "strides"),
    (dict(cache=lambda: rk.KvCache(*(x.transpose(1, 2).contiguous().transpose(1, 2) for x in cache()))), "contiguous"),
    (dict(), "CUDA"),
])
def test_kv_refusals(change, words):
    k, v, s = kv(D=change.get("D", 128), dtype=change.get("dtype", BF))
    c = change["cache"]() if "cache" in change else cache(D=change.get("D", 128))
    s = change.get("slots", s)
    with pytest.raises(ValueError, match=words):
        rk.kv_write(k, v, c, s)
    if "dtype" not in change and "slots" not in change and "D" not in change:
        with pytest.raises(ValueError):
            rk.kv_read(c, s, k, v)


def paged(**kw):
    a = dict(q=torch.zeros(2, 2, 4, 128, dtype=BF), cache=cache(), table=torch.zeros(2, 3, dtype=torch.int32), scale=1.0,
             qpos=torch.zeros(2, 2, dtype=torch.int32), G=2)
    a.update(kw)
    return rk.fmha_paged(a.pop("q"), a.pop("cache"), a.pop("table"), a.pop("scale"), **a)


@pytest.mark.parametrize("kw, words", [
    (dict(q=torch.zeros(2, 2, 4, 96, dtype=BF)), "head dimension"),
    (dict(q=torch.zeros(2, 2, 4, 128)), "bfloat16"),
    (dict(q=torch.zeros(2, 4, 128, dtype=BF)), "B, H, M, D"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), "int32"),
    (dict(table=torch.zeros(3, 3, dtype=torch.int32)), "shape"),
    (dict(qpos=torch.zeros(2, 2)), "int32"),
    (dict(qpos=torch.zeros(2, 1, dtype=torch.int32)), "columns"),
    (dict(G=3), "divide"),
    (dict(G=0), "divide"),
    (dict(prefix_len=3), "without a prefix"),
    (dict(prefix=torch.zeros(2, dtype=torch.int32), prefix_len=33), "2 pages"),
    (dict(prefix=torch.zeros(2, dtype=torch.int32), prefix_len=-1), "2 pages"),
    (dict(prefix=torch.zeros(2, dtype=torch.int64), prefix_len=3), "int32"),
    (dict(out=torch.zeros(2, 2, 4, 128)), "bfloat16"),
    (dict(out=torch.zeros(2, 2, 128, 4, dtype=BF).transpose(2, 3)), "contiguous"),
    (dict(), "CUDA"),
])
def test_paged_refusals(kw, words):
    with pytest.raises(ValueError, match=words):
        paged(**kw)


def delta(**kw):
    T, H, HV, N = 5, 2, 4, 2
    a = dict(q=torch.zeros(T, H, 128, dtype=BF), k=torch.zeros(T, H, 128, dtype=BF), v=torch.zeros(T, HV, 128, dtype=BF),
             g=torch.zeros(T, HV), beta=torch.zeros(T, HV, dtype=BF), cu=torch.tensor([0, 2, 5]), scale=1.0,
             state=torch.zeros(3, HV, 128, 128))
    a.update(kw)
    first = [a.pop(n) for n in ("q", "k", "v", "g", "beta", "cu", "scale", "state")]
    return rk.delta_state(*first, **a)


@pytest.mark.parametrize("kw, words", [
    (dict(v=torch.zeros(5, 3, 128, dtype=BF)), "multiple"),
    (dict(k=torch.zeros(5, 2, 64, dtype=BF)), "shape"),
    (dict(g=torch.zeros(5, 4, dtype=BF)), "float32"),
    (dict(beta=torch.zeros(5, 4)), "bfloat16"),
    (dict(cu=torch.tensor([0, 2, 5], dtype=torch.int32)), "int64"),
    (dict(state=torch.zeros(3, 4, 128, 128, dtype=BF)), "float32"),
    (dict(state=torch.zeros(1, 4, 128, 128)), "slots"),
    (dict(state=torch.zeros(1, 4, 128, 128).expand(3, 4, 128, 128)), "overlap"),
    (dict(state=torch.zeros(3, 128, 4, 128).transpose(1, 2)), "contiguous"),
    (dict(slots=torch.zeros(2, dtype=torch.int64)), "int32"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), "shape"),
    (dict(fresh=torch.zeros(2, dtype=torch.uint8)), "bool"),
    (dict(o=torch.zeros(5, 4, 128)), "bfloat16"),
    (dict(), "CUDA"),
])
def test_delta_refusals(kw, words):
    with pytest.raises(ValueError, match=words):
        delta(**kw)


def test_expanded_outputs_are_refused():
    k, v, s = kv()
    with pytest.raises(ValueError, match="overlap"):
        rk.kv_read(cache(), s, k[:1].expand(4, 2, 128), v)
    one = cache(pages=1)
    with pytest.raises(ValueError, match="overlap"):
        rk.kv_write(k, v, rk.KvCache(*(t.view(torch.uint8).expand(3, *t.shape[1:]).view(t.dtype) for t in one)), s)
    with pytest.raises(ValueError, match="overlap"):
        paged(out=torch.zeros(1, 2, 4, 128, dtype=BF).expand(2, 2, 4, 128))


def test_c_entry_refusals_launch_nothing():
    """Bad sizes, alignment and pointers come back as codes; sizes of zero as success.  No device is touched for the refused ones."""
    lib = abi.load("libreax_decode")
    A = 1 << 20  # a 16-byte aligned address that is never followed

    def write(k=A, ksT=256, kc=A, csP=4096, T=4, H=2, D=128, page=16, pages=3):
        return lib.reax_kv_write(k, ksT, 128, A, 256, 128, kc, A, A, A, csP, 2048, 32, 16, A, T, H, D, page, pages, None)

    assert write(D=64) == -3 and write(page=24) == -2 and write(page=0) == -2 and write(T=-1) == -1 and write(H=0) == -1
    assert write(k=A + 2) == -1 and write(ksT=260) == -1 and write(kc=A + 8) == -1 and write(csP=4100) == -1 and write(k=None) == -1
    assert write(T=0) == 0

    def att(q=A, B=1, H=2, M=4, G=1, D=128, P=2, page=16, Lp=0, prefix=None, table=A, qsM=128, ke=A, ws=A, pages=3):
        return lib.reax_fmha_paged(q, 1024, 512, qsM, A, ke, A, A, 4096, 2048, 32, 16, table, 2, prefix, Lp, A, G, 2, A, 1024, 512,
                                   128, ws, ctypes.c_float(1.0), B, H, M, D, P, page, pages, None)

    assert att(D=100) == -3 and att(page=20) == -2 and att(G=0) == -1 and att(H=0) == -1 and att(P=-1) == -1 and att(Lp=-1) == -1
    assert att(q=A + 4) == -1 and att(qsM=129) == -1 and att(ke=A + 8) == -1 and att(table=None) == -1 and att(Lp=5) == -1
    assert att(P=1 << 30) == -1 and att(P=4096, ws=None) == -5 and att(pages=-1) == -1
    assert att(B=0) == 0 and att(M=0) == 0
    assert lib.reax_fmha_paged_splits(1, 2, 4, 128, 2, 16, 0) == 1
    assert lib.reax_fmha_paged_splits(1, 2, 4, 64, 2, 16, 0) == -3

    def delta(q=A, T=4, S=3, N=2, H=2, HV=4, slots=None, ss=65536, state=A):
        return lib.reax_delta_state(q, A, A, A, A, A, state, ss, slots, None, A, ctypes.c_float(1.0), T, S, N, H, HV, None)

    assert delta(HV=5) == -2 and delta(H=0) == -2 and delta(N=-1) == -1 and delta(T=-1) == -1 and delta(q=None) == -1
    assert delta(q=A + 8) == -1 and delta(state=A + 8) == -1 and delta(ss=65537) == -1 and delta(N=4) == -1
    assert delta(N=0) == 0 and delta(T=0) == 0
