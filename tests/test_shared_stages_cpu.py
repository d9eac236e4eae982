"""The order of waits in the tensor-core kernel of attention over shared positions (csrc/shared_stages.h, csrc/k_shared_tc.cu)
on the CPU: every order of events of its roles, for items of one to five steps after one another. One barrier for all
stages, which lets a loader pass a wait too soon or wait for good, has to be seen failing.
The walk is C++ (tests/shared_stages_check.cpp) built with the host compiler."""
import os
import re
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "transformer-inference-engine_b200", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host C++ compiler")
def test_no_order_of_events_goes_wrong(tmp_path):
    exe = str(tmp_path / "shared_stages_check")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", CSRC,
                    os.path.join(HERE, "shared_stages_check.cpp"), "-o", exe], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.strip() == "ok", p.stdout + p.stderr


def test_the_kernel_takes_its_stages_from_there():
    """A step's end is waited for and told of by the stage's barrier, and a copy waits for the stage's last step."""
    with open(os.path.join(CSRC, "k_shared_tc.cu")) as f:
        source = f.read()
    bars = [line for line in source.splitlines() if "o_full" in line and ("wait_all(" in line or "commit_elected(" in line)]
    assert len(bars) == 2 and all("Stage::of(" in line for line in bars), bars
    assert re.search(r"Stage::used\(step\) && !wait_o\(T::Stage::before\(step\)\)", source)


def test_the_drill_refuses_limits_without_meaning():
    from tie_b200 import MODEL_STATUS, library
    drill = library().tie_attention_shared_wait_drill
    for limit in (0, 2_000_000_001, 1 << 40):
        assert drill(limit) == MODEL_STATUS.index("MODEL_ERR_ARG")
