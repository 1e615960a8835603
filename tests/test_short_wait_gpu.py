"""GPU: the tcgen05 context kernel's bounded waits give up after about a second, with an error status and the CTA's abort
flag, and sit through an arrival that comes late (a probe that includes the same header)."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from hummingbird_b200 import _lib, build

pytestmark = pytest.mark.gpu


class Result(C.Structure):
    _fields_ = [("arrived", C.c_int), ("gave_up", C.c_int), ("after_abort", C.c_int), ("status", C.c_uint),
                ("ns_never", C.c_ulonglong), ("ns_abort", C.c_ulonglong)]


@pytest.fixture(scope="module")
def probe(cuda_lib, tmp_path_factory):
    so = tmp_path_factory.mktemp("short_wait") / "short_wait.so"
    subprocess.run([build.nvcc(), *build.ARCH, "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-I",
                    str(build.CSRC), "-o", str(so), str(Path(__file__).with_name("_short_wait.cu"))], check=True)
    return C.CDLL(str(so))


@pytest.mark.parametrize("sleep", [0, 1])
def test_waits_end_after_about_a_second(probe, sleep):
    r = Result()
    assert probe.short_wait_run(sleep, C.byref(r)) == 0
    assert r.arrived and r.gave_up and r.after_abort and r.status == _lib.HB_ERR_TIMEOUT
    assert 0.25e9 < r.ns_never < 4e9, f"gave up after {r.ns_never / 1e9:.2f} s"
    assert r.ns_abort < 1e6
