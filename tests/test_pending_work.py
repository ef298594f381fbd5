"""Calls that fail after they have launched kernels (csrc/predictor.hip, csrc/class_log_probs.hip), on the CPU: their host code over a runtime that launches
nothing.  Memory that they, or their callers, give back has nothing pending on it."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "arboretum_amd", "csrc")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    sys.path.insert(0, os.path.join(HERE, ".."))
    from arboretum_amd.build import hipcc
    at = tmp_path_factory.mktemp("pending")
    objects = []
    for name in ("predictor", "class_log_probs"):
        objects.append(str(at / (name + ".o")))
        subprocess.check_call([hipcc(), "--offload-arch=gfx950", "--offload-host-only", "-std=c++17", "-O1", "-fPIC", "-x", "hip", "-c",
                               os.path.join(CSRC, name + ".hip"), "-o", objects[-1]])
    out = str(at / "check_pending")
    # (the device code that the host objects name is not there, and nothing asks for it)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-pthread", "-no-pie", "-Wl,--unresolved-symbols=ignore-all", "-D__HIP_PLATFORM_AMD__", "-isystem",
                           "/opt/rocm/include", "-o", out] + objects +
                          ["-x", "c++", os.path.join(CSRC, "staging.hip"), os.path.join(CSRC, "parallel.cpp"), os.path.join(HERE, "native", "check_pending.cpp")])
    return out


@pytest.mark.parametrize("check", ["walk", "labels"])
def test_nothing_is_pending_on_what_is_given_back(program, check):
    r = subprocess.run([program, check], stdout=subprocess.PIPE, timeout=60)
    assert r.returncode == 0, r.stdout.decode()
