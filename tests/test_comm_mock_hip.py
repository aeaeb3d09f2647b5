"""What setting up and leaving an exchange between ranks does to memory (tracking_sdf_amd/csrc/api_comm.cpp), checked
against a stand-in for the HIP runtime that records its calls: no GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tracking_sdf_amd", "csrc")
CASES = ["shm_registers_nothing", "peer_keeps_its_buffer"]


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("comm") / "comm_mock_hip_test")
    p = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Wno-unused-function", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        "-o", out, os.path.join(ROOT, "tests", "host", "comm_mock_hip_test.cpp")] +
                       [os.path.join(CSRC, f) for f in ("api_comm.cpp", "host_util.cpp", "rccl_dyn.cpp")] + ["-ldl", "-pthread", "-lrt"],
                       capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, p.stderr[-4000:]
    return out


@pytest.mark.parametrize("case", CASES)
def test_exchange_set_up_and_end(exe, case):
    p = subprocess.run([exe, case], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stderr[-3000:]
