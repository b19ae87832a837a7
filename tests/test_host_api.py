"""The C ABI's host code under the address and undefined-behaviour sanitizers
(CPU): tests/native/api_check.cpp over aegean-tge_amd/csrc/tge_api.cpp and the
planners, with stand-ins for the HIP runtime and the kernels."""
import os
import shutil
import subprocess

import pytest

from test_host_plan import FLAGS, ROOT

SOURCES = ["aegean-tge_amd/csrc/tge_api.cpp", "aegean-tge_amd/host/plan.cpp", "aegean-tge_amd/host/plan_e4m3.cpp",
           "tests/native/api_check.cpp"]
CXX = "/opt/rocm/llvm/bin/clang++"  # (the sources use _Float16)


@pytest.fixture(scope="module")
def api_check(tmp_path_factory):
    if not shutil.which(CXX):
        pytest.skip("clang++ not available")
    exe = str(tmp_path_factory.mktemp("api") / "api_check")
    cmd = [CXX, *FLAGS, "-I" + os.path.join(ROOT, "tests/native/fake_hip"),
           *[os.path.join(ROOT, s) for s in SOURCES], "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]

    def run(check):
        r = subprocess.run([exe, check], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0 and "api_check ok" in r.stdout, (r.stdout + r.stderr)[-4000:]
    return run


def test_calls_stay_on_their_device(api_check):
    """A call whose plan or pool is on another device is refused, and a batch
    planned anew on another device has its buffers there."""
    api_check("devices")


def test_plan_without_host_memory(api_check):
    """tge_batch_plan returns TGE_ERR_CAPACITY wherever host memory runs out."""
    api_check("memory")
