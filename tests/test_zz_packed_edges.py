"""Packed products at the ends of their types, in every kind of kernel."""
import pytest
import torch

from .packed_shapes import TILES
from .test_gpu_packed import BF16, DEV, F32, INT8
from .test_zz_packed_tiles import _dev_gen, _near, _wide

pytestmark = pytest.mark.gpu

# rows, K, N: streamed, streamed in parts, tiles of 64 x 64, parts of them, 64 x 128, 128 x 256, parts of them
SHAPES = [(3, 256, 200), (20, 9000, 70), (70, 1856, 4258), (300, 9600, 140), (330, 140, 13700), (700, 7680, 8256), (70, 7680, 8256)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_what_is_no_number_stays_in_its_row_and_channel(M, K, N):
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import PackedWeights, product

    g = _dev_gen(M + K)
    x, w = torch.randn((M, K), generator=g, device=DEV), torch.randn((K, N), generator=g, device=DEV)
    clean = product(x, PackedWeights(w))
    bad, broken = x.clone(), w.clone()
    rows, channels = [0, M // 2, M - 1], [1, N // 2, N - 1]
    for r, v in zip(rows, (float("inf"), float("nan"), float("-inf"))):
        bad[r, K - 1 - r % K] = v
    for c, v in zip(channels, (float("nan"), float("-inf"), float("inf"))):
        broken[K - 1 - c % K, c] = v
    want = clean.clone()
    want[rows], want[:, channels] = float("nan"), float("nan")
    packed = PackedWeights(broken)
    got = product(bad, packed)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    # behind a ReLU a NaN is 0, and a gate's own NaN and infinities are the product's
    gate = torch.ones((1, 1, M, N), device=DEV)
    gate[..., 0, 0], gate[..., 1, 1], gate[..., 2, 2] = float("inf"), float("nan"), float("-inf")
    relu = want.nan_to_num().clamp(min=0)
    assert torch.equal(packed_forward(bad.reshape(1, 1, M, K), packed)[0, 0], relu)
    gated, by_hand = packed_forward(bad.reshape(1, 1, M, K), packed, gate=gate)[0, 0], relu * gate[0, 0]
    assert torch.equal(torch.isnan(gated), torch.isnan(by_hand)) and torch.equal(gated.nan_to_num(), by_hand.nan_to_num())
    # bf16: as the sums go; rows and channels of numbers are untouched by those that are not
    clean, got = product(x, PackedWeights(w, dtype=BF16)), product(bad, PackedWeights(broken, dtype=BF16))
    assert not torch.isfinite(got[rows]).any() and not torch.isfinite(got[:, channels]).any()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[rows], keep[:, channels] = False, False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("M", [2, 40, 150, 3000])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_the_largest_sums_fit(M, sign):
    """K = 131072 and 127 everywhere: 127^2 K = 2114060288 of 2^31, in one sum and in parts of it."""
    from burn_dragon_amd.packed import PackedWeights, product

    K, N = 131072, 130
    x, w = torch.full((M, K), 3.0, device=DEV), torch.full((K, N), sign * 0.7, device=DEV)
    x[M // 2] = -3.0
    _near(product(x, PackedWeights(w)), *_wide(x, w, INT8), F32, M)


@pytest.mark.parametrize("M", [1, 40, 300, 3000])
@pytest.mark.parametrize("x_dtype", [F32, BF16])
def test_subnormal_numbers_count(M, x_dtype):
    """bf16: subnormal rows, weights and results are not taken for zeros."""
    from burn_dragon_amd.packed import PackedWeights, product

    K, N = 256, 512
    for row, channel, result in ((2.0**-130, 2.0**100, 2.0**-30), (2.0**100, 2.0**-130, 2.0**-30), (2.0**-70, 2.0**-65, 2.0**-135)):
        x, w = torch.zeros((M, K), device=DEV, dtype=x_dtype), torch.zeros((K, N), device=DEV)
        x[:, 3], w[3] = row, channel
        assert (product(x, PackedWeights(w, dtype=BF16)) == result).all()
    x[:, 3], w[3] = 2.0**-60, 2.0**-70
    assert (product(x, PackedWeights(w, dtype=BF16), out_dtype=BF16) == 2.0**-130).all()


@pytest.mark.parametrize("line", [l for l, k in TILES if l.startswith("grouped") and "tile" in k][::3])
def test_groups_whatever_the_offsets(line):
    """Tiles of groups whose offsets decrease or lie outside: rows of the running maximum, nothing else written."""
    from burn_dragon_amd.packed import PackedWeights, grouped_product

    kind, G, K, N, M = [int(v) for v in line.split()[1:6]]
    kind = INT8 if kind == 2 else BF16
    g = _dev_gen(M)
    x, w = torch.randn((M, K), generator=g, device=DEV), torch.randn((G, K, N), generator=g, device=DEV)
    packed = PackedWeights(w, dtype=kind)
    offsets = torch.randint(-M // 2, M + M // 2, (G + 1,), generator=g, device=DEV).to(torch.int32)
    offsets[0], offsets[G // 2] = -2**31 if G % 2 else 5, 2**31 - 1 if G % 3 == 0 else M // 3
    limits = offsets.cummax(0).values.clamp(0, M).tolist()
    out = grouped_product(x, packed, offsets, out=torch.full((M, N), 7.0, device=DEV))
    for k in range(G):
        if limits[k + 1] > limits[k]:
            _near(out[limits[k]:limits[k + 1]], *_wide(x[limits[k]:limits[k + 1]], w[k], kind), F32, k)
    assert (out[:limits[0]] == 7).all() and (out[limits[-1]:] == 7).all()


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("G,M", [(1000, 16), (3000, 40), (200, 200), (201, 200), (64, 63), (130, 900)])
def test_groups_that_are_mostly_empty(G, M, kind):
    """Every row another group's, all rows the last group's, the first one's, and rows dealt at random."""
    from burn_dragon_amd.packed import PackedWeights, grouped_product

    K, N = 130, 70
    g = _dev_gen(G + M)
    x, w = torch.randn((M, K), generator=g, device=DEV), torch.randn((G, K, N), generator=g, device=DEV)
    packed = PackedWeights(w, dtype=kind)
    spread = torch.zeros(G, dtype=torch.int64)
    spread[torch.randperm(G)[:min(G, M)]] = 1
    spread[G // 2] += M - int(spread.sum())
    ends = {"spread": spread, "last": torch.tensor([0] * (G - 1) + [M]), "first": torch.tensor([M] + [0] * (G - 1)),
            "random": torch.bincount(torch.randint(0, G, (M,), generator=torch.Generator().manual_seed(G)), minlength=G)}
    for name, sizes in ends.items():
        limits = [0, *sizes.cumsum(0).tolist()]
        out = grouped_product(x, packed, torch.tensor(limits, dtype=torch.int32, device=DEV))
        group = torch.repeat_interleave(torch.arange(G), sizes).tolist()
        for k in set(group):
            a, b = limits[k], limits[k + 1]
            _near(out[a:b], *_wide(x[a:b], w[k], kind), F32, (name, k))
