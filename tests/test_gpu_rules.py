"""Penalties, biases and masks on logits (apply_rules) and the counts they read (count_tokens) against numpy in 64 bits.

Tolerance: a division or product, frequency * n, its sum with presence, two subtractions / additions: 5 roundings, each of
at most u = 2^-24 of the magnitudes that pass through it; and the factors n <= 2^24 are exact: 6 u (|z r| + |f| n + |p| + |bias|), magnitudes also
of the negative penalties."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def rules():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device: the GPU tests must run on the MI355X box")
    from burn_dragon_amd import rules as module

    return module


def _reference(logits, seen, newest, rep, pres, freq, bias, allowed):
    z, seen = logits.astype(np.float64), None if seen is None else seen.copy()
    mag = np.abs(z)
    B, V = z.shape
    if seen is not None:
        if newest is not None:
            for b in range(B):
                if 0 <= newest[b] < V:
                    seen[b, newest[b]] += 1
        n = (seen.astype(np.int64) & 0x7FFFFFFF).astype(np.float64)
        r = np.ones((B, 1)) if rep is None else rep.astype(np.float64)[:, None]
        p = np.zeros((B, 1)) if pres is None else pres.astype(np.float64)[:, None]
        f = np.zeros((B, 1)) if freq is None else freq.astype(np.float64)[:, None]
        met = seen != 0
        z = np.where(met, np.where(z > 0, z / r, z * r), z)
        mag = np.abs(z) + np.abs(f) * n + np.abs(p)
        z = z - (f * n + p * (n > 0))
    if bias is not None:
        z = z + bias
        mag = mag + np.abs(np.where(np.isfinite(bias), bias, 0))
    if allowed is not None:
        z = np.where(allowed, z, -np.inf)
    return z, seen, 6 * 2.0**-24 * np.where(np.isfinite(mag), mag, 0)


def _same(got, want, tol):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    ok = np.isfinite(want)
    assert (np.abs(got - want)[ok] <= tol[ok]).all()


@pytest.mark.parametrize("V", [1, 2, 3, 31, 33, 69, 256, 1023, 1024, 1027, 8192, 65601])
@pytest.mark.parametrize("B", [1, 5])
@pytest.mark.parametrize("which", ["penalties", "bias", "mask", "all", "none"])
def test_rules_equal_their_definition(rules, V, B, which):
    rng = np.random.default_rng(V * 10 + B)
    logits = (3 * rng.standard_normal((B, V))).astype(np.float32)
    seen = newest = rep = pres = freq = bias = allowed = None
    if which in ("penalties", "all"):
        seen = rng.integers(0, 5, (B, V)).astype(np.int32) * (rng.random((B, V)) < 0.3)
        seen = np.where(rng.random((B, V)) < 0.2, seen.astype(np.int64) - 2**31, seen).astype(np.int32)
        newest = rng.integers(0, V, B)
        rep, pres, freq = (rng.uniform(lo, hi, B).astype(np.float32) for lo, hi in ((0.7, 1.8), (-0.5, 1), (-0.2, 0.4)))
    if which in ("bias", "all"):
        bias = rng.standard_normal((B, V)).astype(np.float32)
        bias[rng.random((B, V)) < 0.05] = -np.inf
    if which in ("mask", "all"):
        allowed = rng.random((B, V)) < 0.5
        allowed[0] = False  # a row of which nothing is left
    want, seen_want, tol = _reference(logits, seen, newest, rep, pres, freq, bias, allowed)

    def dev(a):
        return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)

    r = rules.LogitRules(dev(rep), dev(pres), dev(freq), dev(bias), None if allowed is None else rules.pack_allowed(dev(allowed)))
    seen_t, logits_t = dev(seen), dev(logits)
    out = rules.apply_rules(logits_t, r, seen_t, dev(newest))
    _same(out, want, tol)
    assert np.array_equal(logits_t.cpu().numpy(), logits)
    if seen is not None:
        assert np.array_equal(seen_t.cpu().numpy(), seen_want)
        seen_t = dev(seen)
    again = rules.apply_rules(logits_t, r, seen_t, dev(newest), out=logits_t)
    assert again is logits_t and torch.equal(again, out)


def test_rows_of_another_tensor_shared_rows_and_scalars(rules):
    rng = np.random.default_rng(5)
    B, T, V = 4, 3, 101
    logits = torch.from_numpy(rng.standard_normal((B, T, V)).astype(np.float32)).to(DEV)
    bias, allowed = rng.standard_normal(V).astype(np.float32), rng.random(V) < 0.6
    seen = (rng.random((B, V)) < 0.3).astype(np.int32)
    r = rules.LogitRules(1.25, None, 0.5, torch.from_numpy(bias).to(DEV), rules.pack_allowed(torch.from_numpy(allowed).to(DEV)))
    out = torch.full((B, 2, V), 7.0, device=DEV)
    rules.apply_rules(logits[:, -1], r, torch.from_numpy(seen).to(DEV), out=out[:, 0])
    want, _, tol = _reference(logits[:, -1].cpu().numpy(), seen, None, np.full(B, 1.25, np.float32), None,
                              np.full(B, 0.5, np.float32), np.tile(bias, (B, 1)), np.tile(allowed, (B, 1)))
    _same(out[:, 0], want, tol)
    assert (out[:, 1] == 7.0).all()


def test_extreme_values_and_ids_outside(rules):
    V = 70
    logits = np.zeros((4, V), np.float32)
    logits[0], logits[1], logits[2], logits[3] = np.nan, np.inf, -np.inf, np.finfo(np.float32).min
    allowed = np.zeros((4, V), bool)
    allowed[:, ::3] = True
    bias = np.where(np.arange(V) % 2, np.inf, -np.inf).astype(np.float32)
    seen = np.zeros((4, V), np.int32)
    seen[:, 5] = 2**31 - 1  # a full count stays full
    newest = np.array([-1, V, 5, 2**40])
    d = lambda a: torch.from_numpy(a).to(DEV)
    seen_t = d(seen)
    r = rules.LogitRules(repetition=2.0, bias=None, allowed=rules.pack_allowed(d(allowed)))
    out = rules.apply_rules(d(logits), r, seen_t, d(newest)).cpu().numpy()
    assert np.isneginf(out[~allowed]).all()  # whatever stood there
    assert np.isnan(out[0][allowed[0]]).all() and np.isposinf(out[1][allowed[1]]).all() and np.isneginf(out[2]).all()
    assert (out[3][allowed[3]] == np.finfo(np.float32).min).all()
    assert np.array_equal(seen_t.cpu().numpy(), seen)
    out = rules.apply_rules(d(logits), rules.LogitRules(bias=d(bias), allowed=rules.pack_allowed(d(allowed)))).cpu().numpy()
    assert np.isneginf(out[~allowed]).all() and np.isnan(out[2][3])


@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (3, 17, 5), (2, 5000, 256), (16, 4001, 8192), (1, 70000, 65601)])
@pytest.mark.parametrize("prompt", [True, False])
def test_counts(rules, B, T, V, prompt):
    rng = np.random.default_rng(T)
    tokens = (V * rng.random((B, T + 3)) ** 2).astype(np.int64)
    tokens[:, ::11] = -1
    tokens[:, 1::13] = V
    lens = rng.integers(-1, T + 5, B).astype(np.int32)
    seen = rng.integers(0, 3, (B, V)).astype(np.int32)
    want = seen.astype(np.int64)
    for b in range(B):
        said = tokens[b, :min(max(int(lens[b]), 0), T)]
        said = said[(said >= 0) & (said < V)]
        if prompt:
            want[b, said] |= -2**31
        else:
            np.add.at(want[b], said, 1)
    seen_t = torch.from_numpy(seen).to(DEV)
    rules.count_tokens(torch.from_numpy(tokens).to(DEV)[:, :T], seen_t, torch.from_numpy(lens).to(DEV), prompt=prompt)
    assert np.array_equal(seen_t.cpu().numpy(), want.astype(np.int32))
    full = torch.zeros((B, V), dtype=torch.int32, device=DEV)
    rules.count_tokens(torch.from_numpy(tokens).to(DEV), full, prompt=False)
    assert int(full.sum()) == int(((tokens >= 0) & (tokens < V)).sum())


def test_a_captured_step_counts_every_replay(rules):
    from burn_dragon_amd import ffi

    ctx = ffi.Context(0)
    B, V = 3, 300
    logits = torch.randn((B, V), device=DEV)
    seen, newest = rules.token_counts(B, V, DEV), torch.zeros((B,), dtype=torch.int64, device=DEV)
    r = rules.LogitRules(1.5, 0.25, 0.125).to(DEV, B)
    out = torch.empty((B, V), device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rules.apply_rules(logits, r, seen, newest, out=out, ctx=ctx)
    eager = rules.token_counts(B, V, DEV)
    for i in range(6):
        newest.copy_(torch.tensor([i % 2, 299, i], device=DEV))
        graph.replay()
        want = rules.apply_rules(logits, r, eager, newest)
        assert torch.equal(out, want) and torch.equal(seen, eager)


def test_full_counts_stay_and_endless_penalties_leave_what_was_not_said(rules):
    tokens = torch.tensor([[0, 1, 1, 1, 2, 3] * 300], device=DEV)
    seen = torch.tensor([[2**31 - 2, -2, 2**30 - 5, -2**31 + 2**30 - 1]], dtype=torch.int32, device=DEV)  # 1, -2: marked, one to go
    rules.count_tokens(tokens, seen)
    assert seen.tolist() == [[2**31 - 1, -1, 2**30 - 5 + 300, -2**31 + 2**30 - 1 + 300]]
    inf = float("inf")
    z = torch.tensor([[1.0, -2.0, 0.5]], device=DEV)
    seen = torch.tensor([[0, -2**31, 3]], dtype=torch.int32, device=DEV)
    out = rules.apply_rules(z, rules.LogitRules(frequency=inf, presence=inf), seen)
    assert out.tolist() == [[1.0, -2.0, -inf]]
