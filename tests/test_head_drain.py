"""CPU: what the lm_head's product kernels wait for after a wait that ran out, in a model of their barriers (head_drain_model.cpp) that
runs the kernels' own arithmetic: whatever warp gives up, and wherever, nothing is on its way when a CTA ends."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_nothing_is_on_its_way_after_a_wait_that_ran_out(tmp_path):
    exe = str(tmp_path / "model")
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(HERE, "..", "rapid_sampling_b200", "csrc"), os.path.join(HERE, "head_drain_model.cpp"),
                    "-o", exe], check=True)
    r = subprocess.run([exe, "20000"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
