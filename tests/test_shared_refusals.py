"""What the operators of many sequences refuse, without a GPU: the C entry points (shared_refusal_test.cpp) and the checks
of the Python functions, which come before a context is asked for."""
import os
import subprocess

import pytest
import torch

from burn_dragon_amd import build
from burn_dragon_amd.rules import LogitRules, apply_rules, count_tokens, pack_allowed, token_counts
from burn_dragon_amd.shared import shared_prefix_attention, shared_prefix_fork
from burn_dragon_amd.slots import copy_slots

HERE = os.path.dirname(os.path.abspath(__file__))


def test_the_c_entry_points_refuse_before_they_touch_a_device(tmp_path):
    exe = str(tmp_path / "shared_refusal_test")
    subprocess.run([build.HIPCC, *build.FLAGS, "-x", "hip", os.path.join(HERE, "shared_refusal_test.cpp"), "-x", "none", "-o", exe,
                    "-L" + build.PKG, "-lbdh_mi355x", "-Wl,-rpath," + build.PKG], check=True, capture_output=True)
    done = subprocess.run([exe], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", (done.returncode, done.stdout, done.stderr)


def _read_args():
    return {"query": torch.zeros(5, 2, 1, 6), "value": torch.zeros(5, 1, 8), "rho": torch.zeros(2, 2, 6, 8),
            "keys": torch.zeros(5, 2, 6, 8), "values": torch.zeros(5, 8, 8), "lens": torch.zeros(5, dtype=torch.int32),
            "freqs": torch.zeros(6), "counts": [3, 2]}


@pytest.mark.parametrize("name,bad", [
    ("query", torch.zeros(5, 2, 1, 6, dtype=torch.float64)), ("query", torch.zeros(5, 2, 1, 12)[..., ::2]),
    ("value", torch.zeros(5, 1, 8, dtype=torch.bfloat16)), ("rho", torch.zeros(2, 2, 6, 8, dtype=torch.float16)),
    ("rho", torch.zeros(2, 2, 5, 8)), ("rho", torch.zeros(2, 2, 8, 6).transpose(2, 3)), ("keys", torch.zeros(5, 2, 7, 8)),
    ("keys", torch.zeros(5, 2, 6, 8, dtype=torch.bfloat16)), ("values", torch.zeros(5, 7, 8)),
    ("lens", torch.zeros(5, dtype=torch.int64)), ("lens", torch.zeros(4, dtype=torch.int32)), ("freqs", torch.zeros(5)),
    ("positions", torch.zeros(5)), ("counts", [3, 3]), ("counts", None), ("counts", [6, -1]), ("counts", [5]),
    ("alibi_slopes", [1.0])])
def test_attention_checks_its_arguments(name, bad):
    args = _read_args()
    args[name] = bad
    with pytest.raises(ValueError):
        shared_prefix_attention(**args)


@pytest.mark.parametrize("name,bad", [
    ("rho", torch.zeros(2, 2, 5, 8)), ("keys", torch.zeros(5, 2, 6, 9)), ("values", torch.zeros(4, 8, 8)),
    ("lens", torch.zeros(5)), ("counts", [1, 1]), ("out", torch.zeros(5, 2, 6, 8, dtype=torch.bfloat16)),
    ("out", torch.zeros(4, 2, 6, 8))])
def test_fork_checks_its_arguments(name, bad):
    args = {k: v for k, v in _read_args().items() if k in ("rho", "keys", "values", "lens", "counts")}
    args[name] = bad
    with pytest.raises(ValueError):
        shared_prefix_fork(**args)


def test_slots_check_their_arguments():
    a, b = torch.zeros(3, 4, 5), torch.zeros(3, 6, 5)
    for buffers, origin in [([(a, b.to(torch.int32), 1)], [0] * 4), ([(a, b, 0)], [0] * 3), ([(a, b, 1), (a, a, 1)], [0] * 4),
                            ([(a, b, 1)], [0] * 5), ([(a, b, 1)], [6, 0, 0, 0]), ([(a, b, 1)], [-3, 0, 0, 0]),
                            ([(a, b.transpose(0, 2).contiguous().transpose(0, 2), 1)], [0] * 4),
                            ([(a, b, 1)], torch.zeros(4, dtype=torch.int64)), ([(a, b[0], 1)], [0] * 4)]:
        with pytest.raises(ValueError):
            copy_slots(buffers, origin)
    copy_slots([], [])


def test_rules_check_their_arguments():
    z, seen = torch.zeros(2, 40), torch.zeros(2, 40, dtype=torch.int32)
    for rules, more in [(LogitRules(repetition=1.1), {}), (LogitRules(), {"newest": torch.zeros(2, dtype=torch.int64)}),
                        (LogitRules(1.1), {"seen": seen.long()}), (LogitRules(1.1), {"seen": seen[:1]}),
                        (LogitRules(1.1), {"seen": seen, "newest": torch.zeros(3, dtype=torch.int64)}),
                        (LogitRules(1.1), {"seen": seen, "newest": torch.zeros(2, dtype=torch.int32)}),
                        (LogitRules(torch.zeros(3)), {"seen": seen}), (LogitRules(bias=torch.zeros(39)), {}),
                        (LogitRules(bias=torch.zeros(3, 40)), {}), (LogitRules(allowed=torch.zeros(2, dtype=torch.int64)), {}),
                        (LogitRules(allowed=torch.zeros(3, dtype=torch.int32)), {}), (LogitRules(), {"out": torch.zeros(2, 41)})]:
        with pytest.raises(ValueError):
            apply_rules(z, rules, **more)
    with pytest.raises(ValueError):
        apply_rules(z.double(), LogitRules())
    with pytest.raises(ValueError):
        apply_rules(torch.zeros(40, 2).t(), LogitRules())
    for tokens, kw in [(torch.zeros(2, 3, dtype=torch.int32), {}), (torch.zeros(3, 3, dtype=torch.int64), {}),
                       (torch.zeros(3, 2, dtype=torch.int64).t(), {}), (torch.zeros(2, 3, dtype=torch.int64), {"lens": torch.zeros(2)})]:
        with pytest.raises(ValueError):
            count_tokens(tokens, seen, **kw)


def test_tensors_in_host_memory_are_refused():
    """The last check before a context is asked for: no address of host memory reaches a kernel."""
    z, seen, toks = torch.zeros(2, 40), torch.zeros(2, 40, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int64)
    args = _read_args()
    fork = {k: v for k, v in args.items() if k in ("rho", "keys", "values", "lens", "counts")}
    for call in (lambda: shared_prefix_attention(**args), lambda: shared_prefix_fork(**fork), lambda: count_tokens(toks, seen),
                 lambda: apply_rules(z, LogitRules(1.5), seen), lambda: copy_slots([(z, z, 0)], [0, 1]),
                 lambda: copy_slots([(z, z, 0)], torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def test_penalties_that_mean_nothing_and_missing_frequencies():
    for r in (0.0, -1.5, float("nan")):
        with pytest.raises(ValueError):
            LogitRules(repetition=r)
    args = _read_args()
    args["freqs"] = None
    with pytest.raises(ValueError):
        shared_prefix_attention(**args)


def test_packed_masks_and_empty_counts():
    mask = torch.rand(3, 70, generator=torch.Generator().manual_seed(1)) < 0.5
    words = pack_allowed(mask)
    assert words.shape == (3, 3) and words.dtype == torch.int32
    for b in range(3):
        for v in range(96):
            assert (int(words[b, v // 32]) >> (v % 32)) & 1 == (int(mask[b, v]) if v < 70 else 0)
    assert not token_counts(2, 9, "cpu").any()


def test_sizes_that_a_call_cannot_carry_are_refused():
    """Sizes of 2^31 and more, of which a C entry point would see the low 32 bits and serve those; tensors without memory."""
    big = 2**32 + 8

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="meta")

    def read(B=1, h=1, T=1, N=2, d=4, S=4, G=1):
        return {"query": empty(B, h, T, N), "value": empty(B, T, d), "rho": empty(G, h, N, d), "keys": empty(B, h, N, S),
                "values": empty(B, S, d), "lens": empty(B, dtype=torch.int32), "freqs": empty(N), "counts": [B]}

    for size in ("B", "h", "T", "N", "d", "S"):
        args = read(**{size: big})
        with pytest.raises(ValueError, match="2\\^31"):
            shared_prefix_attention(**args)
        if size != "T":
            with pytest.raises(ValueError, match="2\\^31"):
                shared_prefix_fork(**{k: v for k, v in args.items() if k in ("rho", "keys", "values", "lens", "counts")})
    with pytest.raises(ValueError, match="2\\^31"):  # N fits, the 2 N rows of PoPE do not
        shared_prefix_attention(**read(N=2**30), rotary_embedding="pope")
    u8 = torch.uint8
    for dst, src, dim in [((big, 2), (big, 3), 1), ((2**16, 2**16, 2, 3), (2**16, 2**16, 2, 3), 2), ((big, 2), (4, 2), 0), ((4, 2), (big, 2), 0)]:
        with pytest.raises(ValueError, match="2\\^31"):
            copy_slots([(empty(*dst, dtype=u8), empty(*src, dtype=u8), dim)], [0] * min(dst[dim], 4))
    for B, V in [(1, big), (big, 1)]:
        seen = empty(B, V, dtype=torch.int32)
        with pytest.raises(ValueError, match="2\\^31"):
            apply_rules(empty(B, V), LogitRules(), seen)
        with pytest.raises(ValueError, match="2\\^31"):
            count_tokens(empty(B, 3, dtype=torch.int64), seen)
    with pytest.raises(ValueError, match="2\\^31"):
        count_tokens(empty(1, big, dtype=torch.int64), empty(1, 9, dtype=torch.int32))


def test_penalties_that_would_make_logits_nan():
    """0 times an infinite repetition, 0 divided by one that f32 rounds to 0, and penalties that are no numbers."""
    for r in (float("inf"), 1e39, 1e-46):
        with pytest.raises(ValueError):
            LogitRules(repetition=r)
    for p in (float("nan"), float("-inf")):
        with pytest.raises(ValueError):
            LogitRules(presence=p)
        with pytest.raises(ValueError):
            LogitRules(frequency=p)
    assert LogitRules(0.5, -1.0, float("inf")).penalises and LogitRules(3, 1, 0).penalises
