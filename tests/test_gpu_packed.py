"""Projections through packed weights against their definitions in 64 bits.

8-bit weights: whole numbers and scales are made here by the rule (each operation rounded to 32 bits) and the sums of products
are exact, so a result is off by its own roundings alone: the sum to f32, two products with scales, and where they are there the
bias, the threshold and the gate; each is half a step, 2^-24 of the value it rounds (2^-8 more for a bf16 result).
bf16 weights: K products are added in f32 in some order, each addition off by at most 2^-23 of the sum of magnitudes (a step, in
case the matrix cores cut instead of rounding)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, INT8 = torch.float32, torch.bfloat16, torch.int8


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def whole_numbers(v, axis):
    """f64 whole numbers and f64 scales (kept axis) of f32 values."""
    v = v.numpy().astype(np.float32)
    top = np.abs(v).max(axis=axis, keepdims=True) if v.shape[axis] else np.zeros(1, np.float32)
    fits = top >= np.float32(2.0**-118)
    with np.errstate(all="ignore"):
        scale = np.where(fits, top / np.float32(127), np.float32(0)).astype(np.float32)
        up = np.where(fits, np.float32(127) / top, np.float32(0)).astype(np.float32)
        q = np.where(fits, np.rint(v * up), 0.0).astype(np.float64)
    bad = ~np.isfinite(top)
    return np.where(bad, 0.0, q), np.where(bad, np.nan, scale).astype(np.float64)


def definition(x, w, kind):
    """x [M,K], w [K,N] as CPU f32 -> result [M,N] in f64 and the bound of its error in f32."""
    if kind is INT8:
        q, s = whole_numbers(x, 1)
        p, t = whole_numbers(w, 0)
        out = (q @ p) * s * t
        return out, 3.1 * 2.0**-24 * np.abs(out)
    a, b = x.to(BF16).double().numpy(), w.to(BF16).double().numpy()
    return a @ b, (x.shape[1] + 1) * 2.0**-23 * (np.abs(a) @ np.abs(b))


def rounded(bound, value, dtype):
    return bound + (2.0**-8 * (np.abs(value) + bound) if dtype is BF16 else 0.0)


def close(got, want, bound, what=""):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    fine = ~np.isnan(want)
    off = np.abs(got - want)[fine] - bound[fine]
    assert off.size == 0 or off.max() <= 0, (what, off.max(), int((off > 0).sum()))


def pack(w, kind, **kw):
    from burn_dragon_amd.packed import PackedWeights

    return PackedWeights(w.to(DEV), dtype=kind, **kw)


def rows_of(g, M, K, dtype):
    """Rows of different magnitudes, one of zeros among them."""
    x = torch.randn((M, K), generator=g) * torch.exp2(torch.randint(-6, 7, (M, 1), generator=g).float())
    if M > 2:
        x[M // 2] = 0.0
    return x.to(dtype).float()


SIZES = [(1, 1, 1), (1, 256, 256), (2, 15, 7), (3, 16, 8), (5, 63, 65), (16, 64, 64), (17, 65, 63), (4, 4096, 72), (33, 100, 200),
         (64, 257, 129), (65, 128, 130), (130, 1000, 66), (200, 512, 321), (1, 32768, 256), (7, 5000, 9), (31, 9000, 40),
         (22, 3201, 203), (51, 1275, 92), (45, 2100, 700), (40, 1100, 17000), (500, 9, 324), (700, 70, 40), (300, 9000, 580), (90, 131072, 33)]


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("x_dtype,out_dtype", [(F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
def test_product(M, K, N, kind, x_dtype, out_dtype):
    from burn_dragon_amd.packed import product

    g = gen(M * 7 + K + N)
    x, w = rows_of(g, M, K, x_dtype), torch.randn((K, N), generator=g) * torch.exp2(torch.randint(-4, 5, (1, N), generator=g).float())
    if N > 3:
        w[:, 2] = 0.0
    want, bound = definition(x, w, kind)
    got = product(x.to(DEV, x_dtype), pack(w, kind), out_dtype=out_dtype)
    assert got.dtype is out_dtype
    close(got, want, rounded(bound, want, out_dtype))


@pytest.mark.parametrize("kind", [INT8, BF16])
def test_weights_in_bf16_pack_as_the_same_values_in_f32(kind):
    from burn_dragon_amd.packed import PackedWeights

    w = torch.randn((2, 70, 33), generator=gen(1)).to(BF16)
    a, b = PackedWeights(w.to(DEV), dtype=kind), PackedWeights(w.float().to(DEV), dtype=kind)
    assert torch.equal(a.data, b.data) and (kind is BF16 or torch.equal(a.scales, b.scales))
    assert a.nbytes == b.nbytes and a.groups == 2


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("M", [1, 40, 150])
def test_rows_with_strides_and_a_place_of_their_own(M, kind):
    """Rows and results inside wider tensors, at places aligned to their values only; what lies between them stays."""
    from burn_dragon_amd.packed import product

    g = gen(M)
    for x_dtype, K in ((F32, 96), (BF16, 96), (BF16, 101)):
        wide = torch.randn((M, K + 5), generator=g).to(x_dtype)
        w = torch.randn((K, 75), generator=g)
        packed = pack(w, kind)
        out = torch.full((M, 90), 7.0, device=DEV)
        got = product(wide.to(DEV)[:, 3:3 + K], packed, out=out[:, 1:76])
        want, bound = definition(wide[:, 3:3 + K].float(), w, kind)
        close(got, want, bound)
        assert (out[:, :1] == 7).all() and (out[:, 76:] == 7).all()
        # columns first: rows that are no rows in memory
        turned = wide[:, 3:3 + K].t().contiguous().to(DEV).t()
        assert torch.equal(product(turned, packed), got)
        assert torch.equal(product(wide[:, 3:3 + K].contiguous().reshape(1, M, 1, K).to(DEV), packed), got.reshape(1, M, 1, 75))


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("B,h,T,d,N", [(1, 4, 1, 256, 256), (4, 4, 1, 256, 256), (3, 2, 5, 33, 70), (2, 3, 70, 64, 130), (1, 1, 1, 1, 1),
                                       (2, 8, 33, 100, 129), (20, 2, 1, 40, 65), (1, 2, 300, 128, 64), (2, 3, 20, 3000, 70),
                                       (3, 2, 50, 4100, 66), (1, 3, 1, 5000, 130)])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("x_dtype,gate_dtype,out_dtype", [(F32, F32, F32), (BF16, BF16, BF16), (F32, None, BF16), (BF16, F32, F32)])
def test_relu_lowrank(B, h, T, d, N, shared, kind, x_dtype, gate_dtype, out_dtype):
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward

    g = gen(B + 10 * h + 100 * T + d + N)
    x = rows_of(g, B * (1 if shared else h) * T, d, x_dtype).reshape(B, 1 if shared else h, T, d)
    w, bias = torch.randn((h, d, N), generator=g), torch.randn((h, 1, N), generator=g)
    gate = None if gate_dtype is None else torch.randn((B, h, T, N), generator=g).to(gate_dtype)
    for with_bias, threshold in ((False, 0.0), (True, 0.3)):
        got = packed_forward(x.to(DEV, x_dtype), pack(w, kind), bias.to(DEV) if with_bias else None, threshold,
                             None if gate is None else gate.to(DEV), out_dtype=out_dtype)
        want, bound = np.empty((B, h, T, N)), np.empty((B, h, T, N))
        for b in range(B):
            for i in range(h):
                s, e = definition(x[b, 0 if shared else i], w[i], kind)
                c = bias[i].double().numpy() if with_bias else 0.0
                thr = float(np.float32(threshold))
                e = e + 2.0**-24 * 1.01 * (np.abs(s + c) + np.abs(s + c - thr)) + 2 * 2.0**-24 * e
                s = s + c - thr
                # below the threshold by more than its error: 0; else off by no more than the sum was
                want[b, i], bound[b, i] = np.maximum(s, 0.0), np.where(s < -e, 0.0, e)
        if gate is not None:
            m = gate.double().numpy()
            bound = np.abs(m) * bound + 1.01 * 2.0**-24 * np.abs(m * want)
            want = want * m
        close(got, want, rounded(bound, want, out_dtype), (with_bias, threshold))


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("sizes,spare", [([3], 0), ([0, 5, 0, 11], 2), ([1] * 9, 0), ([0, 0, 0], 4), ([70, 1, 0, 130, 64], 3), ([200, 0, 1], 0),
                                         ([0] * 70 + [4] + [0] * 80 + [2, 1], 1), ([1, 2] * 100, 7)])
@pytest.mark.parametrize("K,N", [(64, 64), (100, 130), (300, 65)])
def test_grouped_product(sizes, spare, K, N, kind):
    from burn_dragon_amd.packed import grouped_product

    G, first = len(sizes), spare // 2
    limits = [first + s for s in np.cumsum([0] + sizes).tolist()]
    M = limits[-1] + spare - first
    g = gen(G + K)
    x, w = rows_of(g, M, K, F32), torch.randn((G, K, N), generator=g)
    packed = pack(w, kind)
    for x_dtype, out_dtype in ((F32, F32), (BF16, BF16)):
        out = torch.full((M, N), 7.0, device=DEV, dtype=out_dtype)
        xs = x.to(x_dtype)
        got = grouped_product(xs.to(DEV), packed, torch.tensor(limits, device=DEV, dtype=torch.int32), out=out)
        assert got is out
        for k in range(G):
            a, b = limits[k], limits[k + 1]
            if b > a:
                want, bound = definition(xs[a:b].float(), w[k], kind)
                close(got[a:b], want, rounded(bound, want, out_dtype), k)
        assert (got[:limits[0]] == 7).all() and (got[limits[-1]:] == 7).all()
        again = grouped_product(xs.to(DEV), packed, limits, out_dtype=out_dtype)
        assert torch.equal(again[limits[0]:limits[-1]], got[limits[0]:limits[-1]])


@pytest.mark.parametrize("offsets", [[0, 90, 20, 50, 400], [-5, -1, 30, 2**31 - 1, 60], [70, 10, 10, 70, 80], [100, 100, 0, 0, 0],
                                     [-2**31, 2**31 - 1, -2**31, 2**31 - 1, 0]])
@pytest.mark.parametrize("M", [7, 100])
def test_offsets_that_are_none_count_as_their_running_maximum(M, offsets):
    from burn_dragon_amd.packed import grouped_product

    g = gen(3)
    x, w = rows_of(g, M, 64, F32), torch.randn((4, 64, 70), generator=g)
    out = torch.full((M, 70), 7.0, device=DEV)
    got = grouped_product(x.to(DEV), pack(w, INT8), torch.tensor(offsets, device=DEV, dtype=torch.int32), out=out)
    limits = np.clip(np.maximum.accumulate(offsets), 0, M).tolist()
    for k in range(4):
        a, b = limits[k], limits[k + 1]
        if b > a:
            close(got[a:b], *definition(x[a:b], w[k], INT8))
    assert (got[:limits[0]] == 7).all() and (got[limits[-1]:] == 7).all()


@pytest.mark.parametrize("M", [1, 6, 100])
def test_rows_and_channels_that_are_no_numbers(M):
    """8 bits: a row or channel with an infinity or a NaN gives NaN and no other does; bf16: as the sums go."""
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import product

    g = gen(M)
    x, w = rows_of(g, M, 130, F32), torch.randn((130, 70), generator=g)
    x[0, 5] = float("inf")
    w[3, 9], w[129, 69] = float("nan"), float("-inf")
    packed = pack(w, INT8)
    got = product(x.to(DEV), packed)
    close(got, *definition(x, w, INT8))
    assert torch.isnan(got[0]).all() and torch.isnan(got[:, 9]).all() and torch.isnan(got[:, 69]).all()
    zeros = packed_forward(x.reshape(1, 1, M, 130).to(DEV), packed)  # a NaN is not above the threshold
    assert not torch.isnan(zeros).any() and (zeros[0, 0, 0] == 0).all()
    wide = pack(w, BF16)
    got = product(x.to(DEV), wide)
    assert torch.isnan(got[:, 9]).all() and not torch.isfinite(got[0]).any() and (torch.isinf(got[1:, 69]) | torch.isnan(got[1:, 69])).all()


@pytest.mark.parametrize("M", [3, 80])
def test_the_ends_of_the_range_of_f32(M):
    """Magnitudes from below the least that has a scale to the largest: what is too small counts as zeros."""
    from burn_dragon_amd.packed import product

    g = gen(M)
    x, w = torch.randn((M, 96), generator=g).clamp(-3, 3), torch.randn((96, 40), generator=g)
    x[0] *= 2.0**-119 / x[0].abs().max()
    x[1] *= 2.0**-116
    x[2] *= 2.0**126
    w[:, 1] *= 2.0**-130
    got = product(x.to(DEV), pack(w, INT8))
    want, bound = definition(x, w, INT8)
    assert (want[0] == 0).all()
    limit = float(np.finfo(np.float32).max)
    over = np.abs(want) > limit
    got = got.double().cpu().numpy()
    assert np.isinf(got[over]).all()
    # below the normal numbers a rounding is half a subnormal step; (sum s_m) t_n holds its steps where sum s_m is above them
    assert (np.abs(got - np.where(over, 0, want))[~over] <= (bound + 2.0**-149 * (1 + np.abs(w.numpy()).max()))[~over]).all()
    largest = torch.tensor([[3.4e38, -3.4e38, 1.0]])
    plain = product(largest.to(DEV), pack(torch.eye(3), BF16))
    assert torch.isfinite(plain).all() and abs(plain[0, 0].item() / 3.4e38 - 1) <= 2.0**-8


def test_nothing_to_do():
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import grouped_product, product

    w = pack(torch.ones(3, 8, 5), INT8)
    one = pack(torch.ones(8, 5), INT8)
    assert product(torch.zeros(0, 8, device=DEV), one).shape == (0, 5)
    assert product(torch.zeros(2, 0, 8, device=DEV), one).shape == (2, 0, 5)
    assert grouped_product(torch.zeros(0, 8, device=DEV), w, [0, 0, 0, 0]).shape == (0, 5)
    assert packed_forward(torch.zeros(0, 1, 3, 8, device=DEV), w).shape == (0, 3, 3, 5)
    assert packed_forward(torch.zeros(2, 3, 0, 8, device=DEV), w).shape == (2, 3, 0, 5)
    none = pack(torch.ones(0, 8, 5), INT8)
    assert grouped_product(torch.zeros(4, 8, device=DEV), none, [0]).shape == (4, 5)
