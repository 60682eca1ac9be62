"""How exact the products of shared_prefix_attention and shared_prefix_fork are, apart from the length of their sums: `a` numbers of
a sum are not zero, the others are, so what an output may be off by does not grow with the sizes.

Tolerance.  u = 2^-24, and of every product p of two f32 numbers
  * six of the nine products of their bf16 terms are taken: |b - hi| <= 2^-8 |b|, |b - hi - mid| <= 2^-16 |b|, hi + mid + lo = b,
    so mid lo, lo mid and lo lo are at most (2 * 2^-24 + 2^-32) |p| <= 2.1 u |p|; with a bf16 factor, or on the f32 cores,
    nothing is left out;
  * a matrix instruction aligns its addends to the largest and may drop what is below one step of it, 2 u each: the one of the
    leading terms adds at most a products and what was there in each of at most a steps, 2 u (a + a) of their sum; those of the
    other terms are 2^-7 of it and less, five of them 0.16 a u in all;
  * a sum that is put together from parts rounds a - 1 times more, u each: to add a zero is exact.
So |error| <= u (2 + 6 a) * (the sum of the |p|).  One more factor (a score times a value) is rounded once in the product and once
in the sum it goes through."""
import numpy as np
import pytest
import torch

DEV = "cuda:0"
U = 2.0**-24
F32, BF16 = torch.float32, torch.bfloat16


def _bound(a):
    return U * (2 + 6 * a)


def _few(rng, rows, n, a):
    """[rows, n]: a numbers of every row are not zero, none of them small"""
    x = np.zeros((rows, n), np.float32)
    for r in range(rows):
        x[r, rng.choice(n, a, replace=False)] = 0.5 + 2 * rng.random(a)
    return x


def _read_case(seed, B, N, d, a, dtype):
    rng = np.random.default_rng(seed)
    x = _few(rng, B * 2, N, a).reshape(B, 2, N)
    rho = torch.from_numpy(rng.standard_normal((1, 2, N, d)).astype(np.float32)).to(dtype)
    return x, rho


def _terms(x):
    """the three bf16 terms of f32 numbers, as 64-bit numbers"""
    x = torch.from_numpy(np.ascontiguousarray(x, np.float32))
    out = []
    for _ in range(3):
        t = x.to(BF16).to(F32)
        out.append(t.numpy().astype(np.float64))
        x = x - t
    assert not x.any()
    return out


def _product(a, b, pairs):
    ta, tb = _terms(a), _terms(b)
    return sum(ta[i] @ tb[j] for i, j in pairs)


SIX = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]


@pytest.mark.parametrize("a", [1, 4])
def test_the_tolerance_sees_every_lost_term(a):
    """On the host, at the sizes below: the six products are within what the bound leaves for them, and any five are not."""
    x, rho = _read_case(3, 20, 300, 64, a, F32)
    x, rho = x[:, 0], rho[0, 0].numpy()
    want, size = x.astype(np.float64) @ rho, np.abs(x).astype(np.float64) @ np.abs(rho)
    assert (np.abs(_product(x, rho, SIX) - want) <= 2.1 * U * size).all()
    for lost in SIX:
        kept = [p for p in SIX if p != lost]
        assert (np.abs(_product(x, rho, kept) - want) > _bound(a) * size).any(), lost
    half = torch.from_numpy(rho).to(BF16).float().numpy()  # a bf16 state: its terms are (itself, 0, 0)
    want, size = x.astype(np.float64) @ half, np.abs(x).astype(np.float64) @ np.abs(half)
    for lost in range(3):
        kept = [(i, 0) for i in range(3) if i != lost]
        assert (np.abs(_product(x, half, kept) - want) > _bound(a) * size).any(), lost


@pytest.fixture(scope="module")
def shared():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device: the GPU tests must run on the MI355X box")
    from burn_dragon_amd import shared

    return shared


def _call(shared, x, rho, keys, values, lens, B, N, d, T=1):
    return shared.shared_prefix_attention(x, torch.zeros((B, T, d), device=DEV), rho, keys, values, lens, None,
                                          rotary_embedding="alibi", alibi_slopes=[0.0, 0.0])


# sequences, neurons, columns, state: the f32 cores (up to 16 queries), split f32 states (17 and more), bf16 states
SIZES = [(4, 300, 64, F32), (16, 514, 132, F32), (20, 300, 64, F32), (32, 1030, 256, F32), (40, 258, 68, F32), (3, 300, 64, BF16),
         (20, 514, 132, BF16), (40, 300, 512, BF16), (5, 130, 4, BF16)]


@pytest.mark.gpu
@pytest.mark.parametrize("a", [1, 4])
@pytest.mark.parametrize("B,N,d,dtype", SIZES)
def test_products_with_the_prompts_state(shared, B, N, d, dtype, a):
    x, rho = _read_case(3, B, N, d, a, dtype)
    keys, values = torch.zeros((B, 2, N, 4), device=DEV), torch.zeros((B, 4, d), device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    out = _call(shared, torch.from_numpy(x)[:, :, None].to(DEV), rho.to(DEV), keys, values, lens, B, N, d)
    r = rho.double().numpy()[0]
    want, size = np.einsum("bhn,hnd->bhd", x.astype(np.float64), r), np.einsum("bhn,hnd->bhd", np.abs(x), np.abs(r))
    err = np.abs(out[:, :, 0].double().cpu().numpy() - want)
    assert (err <= _bound(a) * size).all(), (err / size).max() / U


# tokens that use other neurons than the tokens before them: their scores are zero.  Few queries, and dense products
@pytest.mark.gpu
@pytest.mark.parametrize("B,T,N,d,dtype", [(2, 7, 300, 64, F32), (3, 9, 514, 132, F32), (3, 9, 514, 132, BF16), (2, 3, 130, 4, BF16),
                                           (6, 8, 4096, 128, F32), (6, 8, 4096, 128, BF16)])
def test_products_of_several_tokens(shared, B, T, N, d, dtype):
    rng = np.random.default_rng(5)
    x = np.zeros((B, 2, T, N), np.float32)
    for b in range(B):
        for h in range(2):
            x[b, h, np.arange(T), rng.choice(N, T, replace=False)] = 0.5 + 2 * rng.random(T)
    rho = torch.from_numpy(rng.standard_normal((1, 2, N, d)).astype(np.float32)).to(dtype)
    keys, values = torch.zeros((B, 2, N, 12), device=DEV), torch.zeros((B, 12, d), device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    out = _call(shared, torch.from_numpy(x).to(DEV), rho.to(DEV), keys, values, lens, B, N, d, T)
    r = rho.double().numpy()[0]
    want = np.einsum("bhtn,hnd->bhtd", x.astype(np.float64), r)
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= _bound(1) * np.abs(want)).all(), (err / (np.abs(want) + 1e-30)).max() / U


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,d,dtype", SIZES)
def test_products_with_own_keys(shared, B, N, d, dtype):
    """A prompt's state of zeros and one token said before: out = (q . k) v, a = 1 product in q . k."""
    rng = np.random.default_rng(7)
    x = _few(rng, B * 2, N, 1).reshape(B, 2, 1, N)
    k = rng.standard_normal((B, 2, N)).astype(np.float32)
    v = rng.standard_normal((B, d)).astype(np.float32)
    keys, values = torch.zeros((B, 2, N, 4), device=DEV), torch.zeros((B, 4, d), device=DEV)
    keys[:, :, :, 0], values[:, 0] = torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV)
    lens = torch.ones(B, dtype=torch.int32, device=DEV)
    out = _call(shared, torch.from_numpy(x).to(DEV), torch.zeros((1, 2, N, d), device=DEV, dtype=dtype), keys, values, lens, B, N, d)
    want = np.einsum("bhn,bhn->bh", x[:, :, 0].astype(np.float64), k)[..., None] * v[:, None].astype(np.float64)
    err = np.abs(out[:, :, 0].double().cpu().numpy() - want)
    assert (err <= (_bound(1) + 2 * U) * np.abs(want)).all(), (err / (np.abs(want) + 1e-30)).max() / U


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 4])
@pytest.mark.parametrize("N,d,S", [(300, 64, 8), (70, 132, 8), (130, 320, 72), (130, 192, 128), (66, 180, 132)])
def test_products_of_a_fork(shared, N, d, S, n):
    """n tokens added to a state of zeros: products of keys and values, in every number of columns and tokens."""
    rng = np.random.default_rng(9)
    B = 3
    keys, values = np.zeros((B, 2, N, S), np.float32), np.zeros((B, S, d), np.float32)
    at = np.sort(rng.choice(S, n, replace=False))  # the others said nothing: keys of zero
    keys[:, :, :, at] = rng.standard_normal((B, 2, N, n))
    values[:] = rng.standard_normal((B, S, d))
    lens = torch.full((B,), S, dtype=torch.int32, device=DEV)
    out = shared.shared_prefix_fork(torch.zeros((1, 2, N, d), device=DEV), torch.from_numpy(keys).to(DEV),
                                    torch.from_numpy(values).to(DEV), lens, rotary_embedding="alibi", alibi_slopes=[0.0, 0.0])
    want, size = (np.einsum("bhns,bsd->bhnd", f(keys[..., at].astype(np.float64)), f(values[:, at].astype(np.float64)))
                  for f in (lambda t: t, np.abs))
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= _bound(n) * size).all(), (err / (size + 1e-30)).max() / U
