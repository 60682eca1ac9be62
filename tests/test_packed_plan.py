"""Packed products on the host, over a stand-in for the HIP runtime (host_runtime.h): no GPU."""
import math
import os
import random
import re
import subprocess

import pytest

from burn_dragon_amd import build

from .packed_shapes import COMPANY, PROMPTS, TILES, prompt_lines

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
    """Lines of packed_plan.cpp -> the kernels that each call launches (with their grids, if asked), and all there are."""
    exe = program(tmp_path_factory.mktemp("plan"), "packed_plan")

    def run(lines, grids=False):
        done = subprocess.run([exe], input="\n".join([*lines, "kernels"]) + "\n", capture_output=True, text=True)
        out = done.stdout.split("\n")
        assert done.returncode == 0 and len(out) > len(lines), done.stderr
        compiled = {k for k in out[len(lines):] if re.match("k_packed|k_prepare_rows|k_row_tops", k)}
        if grids:
            return out[:len(lines)]
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


def _short(kernels):
    return [k.replace(", ", ",").replace("unsigned short", "bf16") for k in kernels]


def test_the_sizes_of_the_tests_take_the_kernels_they_are_for(plan):
    launched, compiled = plan([line for line, _ in TILES])
    assert [(line, " ".join(_short(k))) for (line, _), k in zip(TILES, launched)] == TILES
    ends = {k for k in compiled if re.match(r"k_packed_tile|k_packed_finish|k_packed_few<2, \d, \d, \d, \d, true>", k)}
    assert ends - {k for ks in launched for k in ks} == set()


def test_rows_that_are_compared_take_different_kernels(plan):
    kernels = set()
    for K, N, rows in COMPANY:
        launched = plan([f"product 2 {K} {N} {M} 0 {K} 0 {N}" for M in rows])[0]
        assert len({k for ks in launched for k in ks}) >= len(rows) // 2
        kernels |= {re.sub(r"<2,(\d),.*?((\d+),(\d+),\d,\d)?>", r"\1 \3x\4", k) for ks in launched for k in _short(ks)}
    assert {"k_packed_tile0 64x64", "k_packed_tile0 64x128", "k_packed_tile0 128x256", "k_packed_tile0 256x256", "k_packed_tile3 64x64",
            "k_packed_tile3 128x256"} <= kernels
    assert any(k.startswith("k_packed_few0") for k in kernels) and any(k.startswith("k_packed_few3") for k in kernels)


def test_prompts_of_models_go_through_tiles_and_parts(plan):
    lines = [l for p in PROMPTS for l in prompt_lines(*p)]
    launched = [" ".join(_short(k)) for k in plan(lines)[0]]
    for name, which in (("D_y in tiles for gates", [re.search(r"tile<\d,2,\w+,128,128", k) for k in launched[1::3]]),
                        ("D_y in other tiles", [re.search(r"tile<\d,2,\w+,64,64", k) for k in launched[1::3]]),
                        ("D_y in parts", [re.search(r"finish<\d,2", k) for k in launched[1::3]]),
                        ("D_x in tiles", [re.search(r"tile<\d,1", k) for k in launched[::3]]),
                        ("E in tiles", [re.search(r"tile<\d,0", k) for k in launched[2::3]]),
                        ("E in parts", [re.search(r"finish<\d,0", k) for k in launched[2::3]])):
        assert any(which), name


def test_scales_are_aligned(tmp_path):
    done = subprocess.run([program(tmp_path, "packed_alignment_test")], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", (done.returncode, done.stdout, done.stderr)


def test_groups_without_rows_have_no_workgroups(plan):
    """At most a tile for each whole 16, 32, 64, 128 or 256 rows and one more for each group that can have rows."""
    cases = [(G, M, N) for G in (1, 7, 64, 1000, 65535) for M in (1, 5, 16, 40, 300, 5000) for N in (64, 200)]
    for (G, M, N), line in zip(cases, plan([f"grouped 2 {G} 64 {N} {M} 0 64 0 {N}" for G, M, N in cases], grids=True)):
        kernel, grid = re.match(r"(?:.* \+ )?k_packed_(.*) x(\d+)$", line).groups()
        few = re.match(r"few<2, 0, (\d)", kernel)
        rows, wide = (16 * int(few.group(1)), 64) if few else map(int, re.search(r"(\d+), (\d+), \d, \d>", kernel).groups())
        assert int(grid) == (M // rows + min(M, G)) * -(-N // wide), (G, M, N, line)
