"""Packed products on the host, over a stand-in for the HIP runtime (host_runtime.h): no GPU."""
import os
import subprocess

from burn_dragon_amd import build

HERE = os.path.dirname(os.path.abspath(__file__))


def program(directory, name):
    exe = str(directory / name)
    subprocess.run([build.HIPCC, *build.FLAGS, "-x", "hip", os.path.join(HERE, name + ".cpp"), "-x", "none", "-o", exe,
                    "-L" + build.PKG, "-lbdh_mi355x", "-Wl,-rpath," + build.PKG], check=True, capture_output=True)
    return exe


def test_rows_and_results_may_be_columns_of_one_buffer(tmp_path):
    done = subprocess.run([program(tmp_path, "packed_overlap_test")], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", (done.returncode, done.stdout, done.stderr)
