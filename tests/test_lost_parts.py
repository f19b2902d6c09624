"""What the 8-bit products say where a wait ran out: a part of a split sum that is lost makes its element NaN and no
other (csrc/int8_linear.cu, add_parts_kernel, on buffers of the test's own), and the count of such waits can be read."""

import ctypes
import subprocess

import numpy as np
import pytest

from conftest import PKG, ROOT


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    import rlenv_build

    so = tmp_path_factory.mktemp("parts") / "parts_probe.so"
    cmd = [rlenv_build.nvcc(), *rlenv_build.ARCH, "-O3", "-std=c++17", "--expt-relaxed-constexpr",
           "-shared", "-Xcompiler", "-fPIC", f"-I{ROOT / 'include'}", f"-I{PKG / 'csrc'}",
           str(ROOT / "tests" / "parts_probe.cu"), "-o", str(so)]
    subprocess.run(cmd, check=True, capture_output=True)
    lib = ctypes.CDLL(str(so))
    p, n = ctypes.c_void_p, ctypes.c_longlong
    lib.parts_probe.argtypes = [ctypes.c_int, ctypes.c_int, n, n, p, p, p, p]
    return lib


def test_no_sum_is_taken_for_a_lost_one(probe):
    import int8_linear

    most = int8_linear.MOST_TERMS
    assert -2 ** 31 == probe.parts_probe_lost() < -128 * 127 * most and 128 * 128 * most < 2 ** 31


def test_the_status_is_an_error_code_without_a_device():
    import torch

    import rlenv_lib

    lib, count = rlenv_lib.load(), ctypes.c_uint(7)
    assert lib.int8_linear_status(None, 1) == -1
    if not torch.cuda.is_available():
        assert lib.int8_linear_status(ctypes.byref(count), 1) > 0 and count.value == 0


@pytest.mark.gpu
@pytest.mark.parametrize("floats", [1, 0])
@pytest.mark.parametrize("splits", [1, 2, 8, 16])
def test_a_lost_part_is_nan_and_nothing_else(cuda, probe, floats, splits):
    import torch

    m, f = 37, 61
    g = torch.Generator().manual_seed(splits)
    most = 128 * 128 * 131071 // splits
    parts = torch.randint(-most, most, (splits, m, f), generator=g, dtype=torch.int32)
    lost = torch.rand((m, f), generator=g) < 0.1
    which = torch.randint(0, splits, (m, f), generator=g)
    sums = parts.sum(0, dtype=torch.int64).double().numpy()
    for s in range(splits):
        parts[s][lost & (which == s)] = probe.parts_probe_lost()
    a, w = torch.rand(m, generator=g) + 0.5, torch.rand(f, generator=g) + 0.5
    on = [x.to(cuda) for x in (parts, a, w)]
    out = torch.zeros((m, f), dtype=torch.float32 if floats else torch.bfloat16, device=cuda)
    torch.cuda.synchronize()
    assert probe.parts_probe(floats, splits, m, f, *(x.data_ptr() for x in on), out.data_ptr()) == 0
    got, want = out.double().cpu().numpy(), sums * a.double().numpy()[:, None] * w.double().numpy()
    assert np.array_equal(np.isnan(got), lost.numpy()) and lost.any()
    # the sum's conversion and two products in float32, and the result's own rounding
    tol = (3.1 * 2.0 ** -24 + (0 if floats else 2.0 ** -8)) * abs(want)
    assert (abs(got - want) <= tol)[~lost.numpy()].all()
