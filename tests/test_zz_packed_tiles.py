"""Packed products of more rows than a workgroup streams."""
import pytest
import torch

from .packed_shapes import COMPANY, TILES
from .test_gpu_packed import BF16, DEV, F32, INT8, close, definition, gen, pack, rounded, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("M", [1, 40, 700])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_and_results_in_columns_of_one_buffer(M, dtype, kind):
    from burn_dragon_amd.packed import grouped_product, product

    K, N, g = 128, 200, gen(M)
    x, w = rows_of(g, M, K, dtype), torch.randn((K, N), generator=g)
    packed = pack(w, kind)
    want, bound = definition(x, w, kind)
    for at, to in ((0, K), (N + 5, 3)):
        wide = torch.full((M, K + N + 8), 7.0, device=DEV, dtype=dtype)
        wide[:, at:at + K] = x.to(DEV, dtype)
        before = wide.clone()
        out = product(wide[:, at:at + K], packed, out=wide[:, to:to + N])
        close(out, want, rounded(bound, want, dtype))
        close(grouped_product(wide[:, at:at + K], packed, [0, M], out=wide[:, to:to + N]), want, rounded(bound, want, dtype))
        wide[:, to:to + N] = 7.0
        assert torch.equal(wide, before)
        with pytest.raises(Exception, match="overlaps"):
            product(wide[:, at:at + K], packed, out=wide[:, 8:8 + N])


TYPES = {0: F32, 1: BF16, 2: INT8}


def _whole(v, dim):
    """The rule for 8 bits on the device, each step in 64 bits and rounded to 32: a quotient or product of two numbers of 32 bits that
    is rounded twice so is the one that is rounded once."""
    v = v.double()
    top = v.abs().amax(dim, keepdim=True)
    fits = top >= 2.0**-118
    safe = torch.where(fits, top, torch.ones_like(top))
    once = lambda t: t.float().double()
    zero = torch.zeros_like(top)
    return torch.where(fits, torch.round(once(v * once(127.0 / safe))), zero), torch.where(fits, once(safe / 127.0), zero)


def _wide(x, w, kind):
    """definition() on the device: f32 rows x [M,K] and weights w [K,N] -> the result in 64 bits and its bound."""
    if kind is INT8:
        (q, s), (p, t) = _whole(x, 1), _whole(w, 0)
        out = (q @ p) * s * t
        return out, 3.1 * 2.0**-24 * out.abs()
    a, b = x.to(BF16).double(), w.to(BF16).double()
    return a @ b, (x.shape[1] + 1) * 2.0**-23 * (a.abs() @ b.abs())


def _near(got, want, bound, dtype, what, least=0.0):
    if dtype is BF16:
        bound = bound + 2.0**-8 * (want.abs() + bound)
    off = (got.double() - want).abs() - bound - least
    assert not torch.isnan(got).any() and off.max().item() <= 0, (what, off.max().item(), int((off > 0).sum()))


def _values(g, shape, rows_dim, spread=6):
    """Normal numbers, rows (or channels) of different magnitudes, one of them zeros."""
    scale = [1] * len(shape)
    scale[rows_dim] = shape[rows_dim]
    v = torch.randn(shape, generator=g, device=DEV) * torch.exp2(torch.randint(-spread, spread + 1, scale, generator=g, device=DEV).float())
    v.select(rows_dim, shape[rows_dim] // 2).zero_()
    return v


def _dev_gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _run_product(a, g):
    from burn_dragon_amd.packed import PackedWeights, product

    kind, K, N, M, x_dtype, _, out_dtype, _ = int(a[1]), *[int(v) for v in a[2:]]
    kind, x_dtype, out_dtype = TYPES[kind], TYPES[x_dtype], TYPES[out_dtype]
    x, w = _values(g, (M, K), 0).to(x_dtype), _values(g, (K, N), 1, 4)
    got = product(x, PackedWeights(w, dtype=kind), out_dtype=out_dtype)
    _near(got, *_wide(x.float(), w, kind), out_dtype, a)


def _run_grouped(a, g):
    from burn_dragon_amd.packed import PackedWeights, grouped_product

    kind, G, K, N, M, x_dtype, _, out_dtype, _ = int(a[1]), *[int(v) for v in a[2:]]
    kind, x_dtype, out_dtype = TYPES[kind], TYPES[x_dtype], TYPES[out_dtype]
    x, w = _values(g, (M, K), 0).to(x_dtype), _values(g, (G, K, N), 2, 4)
    # ragged: some groups get nothing, rows before the first and behind the last are nobody's
    cuts = torch.randint(2, M - 3, (G + 1,), generator=g, device=DEV).sort().values
    if G > 2:
        cuts[1 + G // 2] = cuts[G // 2]
    limits = cuts.tolist()
    out = torch.full((M, N), 7.0, device=DEV, dtype=out_dtype)
    got = grouped_product(x, PackedWeights(w, dtype=kind), cuts.to(torch.int32), out=out)
    for k in range(G):
        if limits[k + 1] > limits[k]:
            _near(got[limits[k]:limits[k + 1]], *_wide(x[limits[k]:limits[k + 1]].float(), w[k], kind), out_dtype, (a, k))
    assert (got[:limits[0]] == 7).all() and (got[limits[-1]:] == 7).all()


def _run_lowrank(a, g):
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import PackedWeights

    kind, h, K, N, B, h_in, T, x_dtype, gate_dtype, out_dtype, with_bias = [int(v) for v in a[1:12]]
    threshold, kind, x_dtype, out_dtype = float(a[12]), TYPES[kind], TYPES[x_dtype], TYPES[out_dtype]
    x, w = _values(g, (B * h_in * T, K), 0).reshape(B, h_in, T, K).to(x_dtype), _values(g, (h, K, N), 2, 4)
    bias = torch.randn((h, 1, N), generator=g, device=DEV) if with_bias else None
    gate = None if gate_dtype < 0 else torch.randn((B, h, T, N), generator=g, device=DEV).to(TYPES[gate_dtype])
    got = packed_forward(x, PackedWeights(w, dtype=kind), bias, threshold, gate, out_dtype=out_dtype)
    for i in range(h):
        s, e = _wide(x[:, i if h_in > 1 else 0].reshape(B * T, K).float(), w[i], kind)
        # bias and threshold: a rounding each, and their order's share of the error that is there
        c = 0.0 if bias is None else bias[i].double()
        e = e + 2.0**-24 * 1.01 * ((s + c).abs() + (s + c - threshold).abs()) + 2 * 2.0**-24 * e
        s = s + c - threshold
        e = torch.where(s < -e, torch.zeros_like(e), e)
        s = s.clamp(min=0)
        if gate is not None:
            m = gate[:, i].double().reshape(B * T, N)
            e, s = m.abs() * e + 1.01 * 2.0**-24 * (m * s).abs(), s * m
        _near(got[:, i].reshape(B * T, N), s, e, out_dtype, (a, i))


def test_the_plans_are_those_of_256_cus():
    assert torch.cuda.get_device_properties(0).multi_processor_count == 256


@pytest.mark.parametrize("line,kernels", TILES, ids=[line.replace(" ", "_") for line, _ in TILES])
def test_every_tile(line, kernels):
    a = line.split()
    {"product": _run_product, "grouped": _run_grouped, "lowrank": _run_lowrank}[a[0]](a, _dev_gen(len(line) + sum(map(ord, line))))


@pytest.mark.parametrize("K,N,rows", COMPANY)
def test_a_row_gives_the_same_bits_in_every_kernel(K, N, rows):
    """8 bits: streamed, in tiles of every shape, in parts of k, for scales from 2^-72 to 2^63; and the value is the definition's."""
    from burn_dragon_amd.packed import PackedWeights, product

    g = _dev_gen(K + N)
    x, w = _values(g, (max(rows), K), 0), _values(g, (K, N), 1, 4)
    x[0] *= 2.0**66
    x[5] *= 2.0**-66
    w[:, 3] *= 2.0**-64
    w[:, N - 2] *= 2.0**40
    packed = PackedWeights(w)
    many = product(x, packed)
    # what is subnormal is off by half its least step more, twice where the sum meets the larger scale behind the smaller one
    _near(many, *_wide(x, w, INT8), F32, (K, N), 2.0**-149)
    for M in rows:
        assert torch.equal(product(x[:M], packed), many[:M]), M
        assert torch.equal(product(x[-M:], packed), many[-M:]), M


@pytest.mark.parametrize("kind", [INT8, BF16])
def test_captured_tiles_share_no_workspace(kind):
    """Tiles, tiles of parts, groups and gates, each captured in a graph of its own; replayed with new inputs between eager calls."""
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import PackedWeights, grouped_product, product

    g = _dev_gen(1)
    r = lambda *shape: torch.randn(shape, generator=g, device=DEV)
    w = [PackedWeights(r(*s), dtype=kind) for s in ((1100, 2000), (9000, 140), (3, 600, 700), (2, 256, 1030))]
    offsets = torch.tensor([0, 100, 100, 640], dtype=torch.int32, device=DEV)
    gate = r(2, 2, 500, 1030)
    calls = [(r(700, 1100), lambda x: product(x, w[0])), (r(150, 9000), lambda x: product(x, w[1])),
             (r(700, 600), lambda x: grouped_product(x, w[2], offsets)[:640]), (r(2, 2, 500, 256), lambda x: packed_forward(x, w[3], gate=gate))]
    graphs = []
    for x, call in calls:
        call(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(x)
        graphs.append((graph, out))
    for turn in range(4):
        for (x, _), (graph, _) in zip(calls, graphs):
            x.copy_(r(*x.shape))
            graph.replay()
        torch.cuda.synchronize()
        big = r(2000, 1100)
        product(big, w[0])
        for k, ((x, call), (_, out)) in enumerate(zip(calls, graphs)):
            first = call(x)
            assert torch.equal(first, out), (turn, k)
            assert torch.equal(first, call(x))
