"""The shared-prefix kernel's pipeline gives up, unwinds and reports.

libreax_decode is rebuilt here with the wait limit cut to 300 cycles and waits that poll, so that every wait for a tile's copy,
or for what is made of it, runs out.  The roles must then unwind as built: the abort flag stops
the others at their next wait, the copying warp waits for every copy it armed, the issuing warp for every MMA, tensor memory
is released and the CTAs exit.  Checked: the launch returns, the status word holds the timeout code (and reading clears it), the
rows that were not computed are NaN, and the same context then computes correctly with the normal build.  No fault and no
hang is involved: only bounded waits run out."""
import ctypes
import os
import shutil
import subprocess
import tempfile

import pytest
import torch

from reax_engine_kernels_b200 import abi
from reax_engine_kernels_b200 import build as B
from reax_engine_kernels_b200 import kernels as rk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def short_limit():
    nvcc = shutil.which("nvcc") or B.NVCC
    with tempfile.TemporaryDirectory() as td:
        so = os.path.join(td, "libreax_decode_shortwait.so")
        cmd = ([nvcc] + B.ARCH + B.NVCC_FLAGS + ["-DREAX_WAIT_LIMIT=(300ll)", "-DREAX_WAIT_POLL",
                                                  os.path.join(B.CSRC, "decode_lib.cu"), "-o", so])
        subprocess.run(cmd, check=True, capture_output=True)
        lib = ctypes.CDLL(so)
        for fn, (res, args) in abi.PROTOTYPES["libreax_decode"].items():
            f = getattr(lib, fn)
            f.restype, f.argtypes = res, args
        yield lib


@pytest.mark.parametrize("D", [128, 256])
def test_prefix_pipeline_gives_up_and_context_survives(short_limit, D):
    B_, H, M, page, Lp = 16, 4, 8, 64, 4096
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    c = rk.kv_cache(Lp // page, H, page, D)
    n = Lp
    x, y = (torch.randn(n, H, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    rk.kv_write(x, y, c, torch.arange(n, device="cuda"))
    q = torch.randn(B_, H, M, D, generator=g, device="cuda").bfloat16()
    qpos = torch.full((B_, M), Lp - 1, dtype=torch.int32, device="cuda")
    prefix = torch.arange(Lp // page, dtype=torch.int32, device="cuda")
    none = torch.zeros(B_, 0, dtype=torch.int32, device="cuda")
    good = rk.fmha_paged(q, c, none, D ** -0.5, qpos=qpos, prefix=prefix, prefix_len=Lp)
    assert rk.status("libreax_decode") == 0

    out = torch.zeros_like(q)
    splits = short_limit.reax_fmha_paged_splits(B_, H, M, D, 0, page, Lp)
    ws = torch.zeros(splits * B_ * H * M * (D + 1), device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    k, ke, v, ve = c
    rc = short_limit.reax_fmha_paged(
        q.data_ptr(), *q.stride()[:3], k.data_ptr(), ke.data_ptr(), v.data_ptr(), ve.data_ptr(), k.stride(0), k.stride(1), ke.stride(0),
        ke.stride(1), None, 0, prefix.data_ptr(), Lp, qpos.data_ptr(), 1, qpos.stride(0), out.data_ptr(), *out.stride()[:3], ws.data_ptr(),
        D ** -0.5, B_, H, M, D, 0, page, k.shape[0], st)
    assert rc == 0
    torch.cuda.synchronize()  # the launch ends: no hang
    assert short_limit.reax_b200_status(st) == 0x201
    assert short_limit.reax_b200_status(st) == 0  # read and cleared
    assert torch.isnan(out).any()
    ok = ~torch.isnan(out).any(-1)
    assert torch.equal(out[ok], good[ok])  # a row is computed whole or not at all

    again = rk.fmha_paged(q, c, none, D ** -0.5, qpos=qpos, prefix=prefix, prefix_len=Lp)
    assert rk.status("libreax_decode") == 0 and torch.equal(again, good)
