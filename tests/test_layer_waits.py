"""The bounded waits of the decoder-layer kernels: calls leave the data status
clear, and a wait that runs out sets its timeout bit and lets the kernel end.

The second is shown on libraries built here from the same sources with a limit
of no polls for one kind of wait, which therefore runs out at once; all other
waits keep their limit, so that copies in flight still land before a CTA ends."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess
import types

import pytest
import torch

import build
from rans_vectoradd import _C, fp8_linear, kv4
from rans_vectoradd._lib import DATA_TIMEOUT, LIB


def variant(tmp_path_factory, source: str, define: str) -> ctypes.CDLL:
    """`source` with `define`, and host.cpp, as a library of its own."""
    tmp = tmp_path_factory.mktemp("variant")
    cxx, out = shutil.which("g++") or "g++", str(tmp / "variant.so")
    nvcc = [os.path.join(build.cuda_home(), "bin", "nvcc"), *build.ARCH, "-O3", "-std=c++17", "-Xcompiler", "-fPIC,-fopenmp",
            "-ccbin", cxx, "-diag-suppress", "186"]
    subprocess.run([*nvcc, "-shared", f"-D{define}", os.path.join(build.CSRC, source), build.HOST_SOURCE, "-o", out,
                    "-lgomp", "-cudart", "shared"], check=True, capture_output=True)
    return ctypes.CDLL(out)


def operands(m, n, k, dev):
    g = torch.Generator(device=dev).manual_seed(m)
    x8, w8 = ((torch.randn(r, k, device=dev, generator=g) * 50).to(torch.float8_e4m3fn).view(torch.uint8) for r in (m, n))
    return x8, torch.ones(m, device=dev), w8, torch.full((n,), 0.01, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 5120, 1024), (48, 640, 5120), (129, 12700, 512), (2000, 5121, 400), (1500, 5120, 256)])
def test_linear_leaves_the_status_clear(cuda, m, n, k):
    _C.data_status()
    fp8_linear.linear(*operands(m, n, k, cuda))
    assert _C.data_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(129, 12700, 512), (700, 12700, 2064)])  # one tile a pair, several
def test_linear_reports_a_wait_of_its_epilogue_that_ran_out(cuda, tmp_path_factory, m, n, k):
    lib = variant(tmp_path_factory, "linear.cu", "TANS_B200_EPILOGUE_POLLS=0")
    lib.tans_b200_linear.argtypes = LIB.tans_b200_linear.argtypes
    x8, xs, w8, ws = operands(m, n, k, cuda)
    want = fp8_linear.linear(x8, xs, w8, ws)
    y, status = torch.zeros_like(want), torch.zeros(1, dtype=torch.int32, device=cuda)
    rc = lib.tans_b200_linear(x8.data_ptr(), xs.data_ptr(), w8.data_ptr(), ws.data_ptr(), None, 0, None, None, y.data_ptr(),
                              m, n, k, 0, status.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert status.item() == DATA_TIMEOUT
    # and the device goes on
    _C.data_status()
    assert torch.equal(fp8_linear.linear(x8, xs, w8, ws), want) and _C.data_status() == 0


@pytest.fixture(scope="module")
def no_copy_polls(tmp_path_factory):
    lib = variant(tmp_path_factory, "kv4.cu", "TANS_B200_COPY_POLLS=0")
    lib.tans_b200_kv4_attention.argtypes = LIB.tans_b200_kv4_attention.argtypes
    return types.SimpleNamespace(tans_b200_kv4_attention=lib.tans_b200_kv4_attention,
                                 tans_b200_kv4_attention_workspace_bytes=LIB.tans_b200_kv4_attention_workspace_bytes)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [4, 16])  # tiles of 8 rows and of 16
@pytest.mark.parametrize("lens", [[400, 1, 130], [9000, 3000]])  # the keys of a tile in one CTA, and cut
def test_attention_reports_a_wait_for_copies_that_ran_out(cuda, monkeypatch, no_copy_polls, dim, group, lens):
    page, counts = 64, [-(-n // 64) for n in lens]
    cache = kv4.KV4Cache.allocate(sum(counts), 2, page, dim, cuda)
    for t in (cache.k_codes, cache.v_codes):
        t.random_(0, 256)
    for t in (cache.k_scales, cache.v_scales):
        t.fill_(0x30)
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32, device=cuda)
    for b, c in enumerate(counts):
        table[b, :c] = torch.arange(c) + sum(counts[:b])
    n = torch.tensor(lens, dtype=torch.int32, device=cuda)
    q = torch.randn(len(lens), 2 * group, dim, device=cuda).to(torch.bfloat16)
    _C.data_status()
    want = kv4.attention(cache, q, table, n)
    assert _C.data_status() == 0
    with monkeypatch.context() as m:
        m.setattr(kv4, "LIB", no_copy_polls)
        kv4.attention(cache, q, table, n)
        assert _C.data_status() == DATA_TIMEOUT
    assert torch.equal(kv4.attention(cache, q, table, n), want) and _C.data_status() == 0
