"""What the packed projections refuse, without a GPU: the C entry points (packed_refusal_test.cpp) and the checks of the Python
functions, which come before a context is asked for."""
import os
import subprocess
from types import SimpleNamespace

import pytest
import torch

from burn_dragon_amd import build
from burn_dragon_amd.kernel.relu_lowrank import packed_forward
from burn_dragon_amd.packed import PackedWeights, grouped_product, product

HERE = os.path.dirname(os.path.abspath(__file__))


def test_the_c_entry_points_refuse_before_they_touch_a_device(tmp_path):
    exe = str(tmp_path / "packed_refusal_test")
    subprocess.run([build.HIPCC, *build.FLAGS, "-x", "hip", os.path.join(HERE, "packed_refusal_test.cpp"), "-x", "none", "-o", exe,
                    "-L" + build.PKG, "-lbdh_mi355x", "-Wl,-rpath," + build.PKG], check=True, capture_output=True)
    done = subprocess.run([exe], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", (done.returncode, done.stdout, done.stderr)


@pytest.mark.parametrize("weight", [torch.zeros(4), torch.zeros(1, 2, 3, 4), torch.zeros(4, 4, dtype=torch.float16), torch.zeros(4, 4).t()[:, ::2],
                                    torch.zeros(8, 4).t(), torch.zeros(0, 4), torch.zeros(4, 0), torch.zeros(131073, 1),
                                    torch.zeros(1, 1).expand(4, 4)])
def test_weights_are_checked(weight):
    with pytest.raises(ValueError):
        PackedWeights(weight)


def test_types_of_weights_are_checked():
    for dtype in (torch.float32, torch.uint8, torch.float16):
        with pytest.raises(ValueError):
            PackedWeights(torch.zeros(4, 4), dtype=dtype)


def _weights(groups=3, inner=8, outer=5, on=-1):
    return SimpleNamespace(groups=groups, inner=inner, outer=outer, on=on, few=64, device=torch.device("cpu"))


@pytest.mark.parametrize("x", [torch.zeros(4, 7), torch.zeros(4, 8, dtype=torch.float64), torch.zeros(4, 8, dtype=torch.int8), torch.zeros(())])
def test_rows_are_checked(x):
    with pytest.raises(ValueError):
        product(x, _weights(1))


def test_a_product_takes_weights_of_one_group():
    with pytest.raises(ValueError, match="groups"):
        product(torch.zeros(4, 8), _weights(2))


@pytest.mark.parametrize("offsets", [[0, 1, 2], [0, 1, 2, 3, 4], [0, 3, 2, 4], [-1, 0, 0, 0], [0, 0, 0, 5], torch.zeros(4), torch.zeros(3, dtype=torch.int32),
                                     torch.zeros(4, dtype=torch.int64), torch.zeros(8, dtype=torch.int32)[::2]])
def test_offsets_are_checked(offsets):
    with pytest.raises(ValueError):
        grouped_product(torch.zeros(4, 8), _weights(), offsets)


@pytest.mark.parametrize("name,bad", [
    ("input", torch.zeros(2, 2, 3, 8)), ("input", torch.zeros(2, 3, 8)), ("input", torch.zeros(2, 1, 3, 7)), ("input", torch.zeros(2, 1, 8, 3).transpose(2, 3)),
    ("input", torch.zeros(2, 1, 3, 8, dtype=torch.float16)), ("bias", torch.zeros(3, 4)), ("bias", torch.zeros(3, 5, dtype=torch.bfloat16)),
    ("bias", torch.zeros(5, 3).t()), ("gate", torch.zeros(2, 3, 3, 4)), ("gate", torch.zeros(2, 3, 3, 5, dtype=torch.float64)),
    ("gate", torch.zeros(2, 3, 5, 3).transpose(2, 3))])
def test_lowrank_arguments_are_checked(name, bad):
    args = {"input": torch.zeros(2, 1, 3, 8), name: bad}
    with pytest.raises(ValueError):
        packed_forward(args.pop("input"), _weights(), **args)


def test_tensors_in_host_memory_are_refused():
    """The last check before a context is asked for: no address of host memory reaches a kernel."""
    for call in (lambda: product(torch.zeros(4, 8), _weights(1)), lambda: grouped_product(torch.zeros(4, 8), _weights(), torch.zeros(4, dtype=torch.int32)),
                 lambda: grouped_product(torch.zeros(4, 8), _weights(), [0, 1, 2, 4]), lambda: packed_forward(torch.zeros(2, 3, 1, 8), _weights()),
                 lambda: PackedWeights(torch.zeros(4, 4))):
        with pytest.raises(ValueError, match="HIP device"):
            call()
