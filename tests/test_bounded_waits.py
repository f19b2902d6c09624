"""The bounded wait of the gated block's kernel (csrc/blackwell.cuh): it gives up on a barrier that nothing
arrives at, and time in which the GPU ran something else does not count. The probe is compiled here from
tests/wait_probe.cu; it starts no copy and no matrix product."""

import ctypes
import subprocess

import numpy as np
import pytest

from conftest import PKG, ROOT

MS = 1_000_000
LIMIT = 2000 * MS


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    import rlenv_build

    so = tmp_path_factory.mktemp("waits") / "wait_probe.so"
    cmd = [rlenv_build.nvcc(), *rlenv_build.ARCH, "-O3", "-std=c++17", "--expt-relaxed-constexpr",
           "-shared", "-Xcompiler", "-fPIC", f"-I{ROOT / 'include'}", f"-I{PKG / 'csrc'}",
           str(ROOT / "tests" / "wait_probe.cu"), "-o", str(so)]
    subprocess.run(cmd, check=True, capture_output=True)
    lib = ctypes.CDLL(str(so))
    lib.wait_probe.argtypes = [ctypes.c_uint64, ctypes.c_void_p]
    lib.patience_probe.argtypes = [ctypes.c_uint64, ctypes.c_uint64, ctypes.c_void_p, ctypes.c_int]
    return lib


def over(probe, looks, start=10 ** 12):
    looks = np.asarray(looks, np.uint64) + np.uint64(start)
    return probe.patience_probe(LIMIT, start, looks.ctypes.data, len(looks))


def test_a_wait_is_over_after_its_time(probe):
    looks = np.arange(1, 3001) * MS
    assert over(probe, looks) == 2000  # the first look past two seconds
    assert over(probe, looks[:2000]) == -1
    assert over(probe, looks // 10) == -1


def test_time_without_looks_does_not_count(probe):
    """Three seconds in which another process had the GPU, then the arrival comes soon; and a GPU shared for good
    still gives up."""
    assert over(probe, [MS, 2 * MS, 3002 * MS, 3003 * MS]) == -1
    assert over(probe, 3000 * MS + np.arange(1, 1000) * MS) == -1
    assert over(probe, np.arange(1, 400) * 100 * MS) == 200


def test_the_status_is_an_error_code_without_a_device():
    import torch

    import rlenv_lib

    if torch.cuda.is_available():
        pytest.skip("this is the no-device path")
    lib, count = rlenv_lib.load(), ctypes.c_uint(7)
    assert lib.gated_ffn_status(None, 1) == -1
    assert lib.gated_ffn_status(ctypes.byref(count), 1) > 0 and count.value == 0


@pytest.mark.gpu
def test_a_wait_gives_up(cuda, probe):
    import torch

    out = torch.zeros((32, 6), dtype=torch.int64, device=cuda)
    assert probe.wait_probe(20 * MS, out.data_ptr()) == 0
    first, second, third, flag, took, after = out.cpu().unbind(1)
    assert not first.any() and (flag == 1).all(), "nothing arrives: the wait runs out and says so"
    assert (took >= 20 * MS).all() and (took < 2000 * MS).all()
    assert not second.any() and (after < 1000 * MS).all(), "the next wait, of up to 20 s, gives up at the flag"
    assert third.all(), "an arrival ends a wait"


@pytest.mark.gpu
def test_a_wait_that_ran_out_is_counted(cuda, probe):
    import torch

    out, count = torch.zeros((32, 6), dtype=torch.int64, device=cuda), ctypes.c_uint(7)
    assert probe.wait_probe_status(ctypes.byref(count), 1) == 0
    for runs in (1, 2):
        assert probe.wait_probe(MS, out.data_ptr()) == 0
        assert probe.wait_probe_status(ctypes.byref(count), 0) == 0 and count.value == runs
    assert probe.wait_probe_status(ctypes.byref(count), 1) == 0 and count.value == 2
    assert probe.wait_probe_status(ctypes.byref(count), 0) == 0 and count.value == 0


@pytest.mark.gpu
def test_the_blocks_calls_report_no_wait_that_ran_out(cuda):
    import torch

    import gated_ffn

    gated_ffn.gave_up()
    x, w = torch.randn((700, 96), device=cuda), torch.randn((96, 200), device=cuda)
    y = gated_ffn.forward(x, w, w)
    gated_ffn.backward(y, x, w, w)
    assert gated_ffn.gave_up() == 0 and gated_ffn.gave_up(cuda, clear=False) == 0
