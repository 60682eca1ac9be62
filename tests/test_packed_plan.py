"""Packed products on the host, over a stand-in for the HIP runtime (host_runtime.h): no GPU."""
import math
import os
import random
import re
import subprocess

import pytest

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


INT8, BF16, F32 = 2, 1, 0


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """Lines of packed_plan.cpp -> the kernels that each call launches, and all there are."""
    exe = program(tmp_path_factory.mktemp("plan"), "packed_plan")

    def run(lines):
        done = subprocess.run([exe], input="\n".join([*lines, "kernels"]) + "\n", capture_output=True, text=True)
        out = done.stdout.split("\n")
        assert done.returncode == 0 and len(out) > len(lines), done.stderr
        compiled = {k for k in out[len(lines):] if re.match("k_packed|k_prepare_rows|k_row_tops", k)}
        return [l if l.startswith("refused") else [re.sub(r" x\d+$", "", k) for k in l.split(" + ")] for l in out[:len(lines)]], compiled

    return run


def _calls(n):
    """Calls of all kinds, sizes over their logarithm, half of them whole blocks."""
    rng = random.Random(1)
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    lines = []
    while len(lines) < n:
        kind, t, x, out = rng.choice(["product", "grouped", "lowrank", "lowrank"]), rng.choice([BF16, INT8]), rng.choice([F32, BF16]), rng.choice([F32, BF16])
        K, N, M = log(1, 131072), log(1, 70000), log(1, 20000)
        if rng.random() < 0.5:
            K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
        if kind == "lowrank":
            h, T = rng.choice([1, 2, 3, 4, 8, 64]), rng.choice([1, log(1, 3000)])
            B = max(1, M // T)
            if B * T * h * N > 2**31:
                continue
            lines.append(f"lowrank {t} {h} {K} {N} {B} {rng.choice([1, h])} {T} {x} {rng.choice([-1, 0, 1])} {out} {rng.choice([0, 1])} {rng.choice([0, 0, 0.5])}")
        else:
            if M * N > 2**31:
                continue
            lines.append(f"{kind} {t} {'' if kind == 'product' else log(1, 300)} {K} {N} {M} {x} {K} {out} {N}")
    return lines


def test_every_kernel_is_reached(plan):
    lines = _calls(300000)
    launched, compiled = plan(lines)
    assert not [l for l, k in zip(lines, launched) if isinstance(k, str)]
    assert compiled - {k for ks in launched for k in ks} == set()


def test_what_comes_behind_the_sums_is_the_calls(plan):
    """The last kernel of a call is compiled for what the call asks: 0 scales, 1 ReLU, 2 bias, threshold, ReLU and gate."""
    lines = _calls(100000)
    for line, kernels in zip(lines, plan(lines)[0]):
        behind = int(re.match(r"k_packed_\w+<\d, (\d),", kernels[-1]).group(1))
        a = line.split()
        want = 0 if a[0] != "lowrank" else 2 if a[9] != "-1" or a[11] == "1" or float(a[12]) else 1
        assert behind == want, (line, kernels)
