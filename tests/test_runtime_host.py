"""The runtime's host logic (runtime.cu) over a fake CUDA runtime with two devices (no GPU needed)."""
import subprocess
from pathlib import Path

import pytest

from conftest import ROOT

NATIVE = Path(__file__).resolve().parent / "native"


def build(folder):
    from nx_vulkan_b200 import build as b
    exe = folder / "runtime_test"
    include = Path(b.nvcc()).resolve().parents[1] / "include"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-pthread", f"-I{b.CSRC}", f"-isystem{include}", "-o", str(exe),
                    "-x", "c++", str(b.CSRC / "runtime.cu"), str(NATIVE / "fake_cudart.cpp"),
                    str(NATIVE / "runtime_test.cpp")], check=True, cwd=ROOT)
    return exe


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    return build(tmp_path_factory.mktemp("runtime"))


def holds(exe, name):
    p = subprocess.run([str(exe), name], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout + p.stderr


@pytest.mark.parametrize("name", ["init_default_has_wait_flag", "init_devices_has_wait_flag"])
def test_every_way_to_initialise_has_a_wait_flag(exe, name):
    """The tensor-core cross entropy reports a wait that ran out there: without it, it would write to address 0."""
    holds(exe, name)


@pytest.mark.parametrize("name", ["wait_report_is_its_devices", "wait_report_reaches_every_thread"])
def test_a_wait_that_ran_out_is_told_to_whom_it_concerns(exe, name):
    """The word that the kernel writes is written here by the test: no wait runs out."""
    holds(exe, name)


@pytest.mark.parametrize("name", ["failed_scratch_is_its_call_s", "failed_call_is_its_call_s"])
def test_an_error_is_not_the_next_call_s(exe, name):
    """A workspace that does not fit, a CUDA call that fails: the valid call after it is not refused for it."""
    holds(exe, name)
