"""Buffers that calls share and that captured calls hold, without a GPU (captured_scratch_test.cpp)."""
import os
import subprocess

from burn_dragon_amd import build

HERE = os.path.dirname(os.path.abspath(__file__))


def test_what_a_captured_call_was_given_stays(tmp_path):
    exe = str(tmp_path / "captured_scratch_test")
    subprocess.run([build.HIPCC, *build.FLAGS, "-x", "hip", os.path.join(HERE, "captured_scratch_test.cpp"), "-x", "none", "-o", exe,
                    "-L" + build.PKG, "-lbdh_mi355x", "-Wl,-rpath," + build.PKG], check=True, capture_output=True)
    done = subprocess.run([exe], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", (done.returncode, done.stdout, done.stderr)
