"""Slots of a batch's buffers moved in one launch (copy_slots): every byte equal to indexing, in place and elsewhere."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def slots():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device: the GPU tests must run on the MI355X box")
    from burn_dragon_amd import slots as module

    return module


def _buffers(gen, m):
    """A state of 3 layers, stamps, keys of an odd width, bf16 rows of an odd length, flags, positions."""
    def f(*s, dtype=torch.float32):
        return torch.randn(s, device=DEV, generator=gen).to(dtype)

    return [(f(3, m, 2, 24, 8), 1), (torch.randint(0, 99, (3, m, 2, 24), device=DEV, generator=gen, dtype=torch.int32), 1),
            (f(m, 2, 7, 5), 0), (f(2, m, 33, dtype=torch.bfloat16), 1), (torch.randint(0, 2, (m, 13), device=DEV, generator=gen).bool(), 0),
            (torch.randint(0, 99, (m,), device=DEV, generator=gen, dtype=torch.int32), 0),
            (f(1, m, 70001), 1)]


def _want(dst, src, dim, origin):
    out = dst.clone()
    for i, o in enumerate(origin):
        if o == -1:
            out.select(dim, i).zero_()
        elif 0 <= o < src.shape[dim]:
            out.select(dim, i).copy_(src.select(dim, o))
    return out


IN_PLACE = {
    "identity": lambda n, rng: list(range(n)),
    "cycle": lambda n, rng: [(i + 1) % n for i in range(n)],
    "permutation": lambda n, rng: rng.permutation(n).tolist(),
    "fork": lambda n, rng: [0] * n,
    "beams": lambda n, rng: rng.integers(0, n, n).tolist(),
    "compact": lambda n, rng: sorted(rng.permutation(n)[: (n + 1) // 2].tolist()) + [-1] * (n // 2),
    "free": lambda n, rng: [-1] * n,
    "keep": lambda n, rng: [-2] * n,
    "mixed": lambda n, rng: rng.integers(-2, n, n).tolist(),
}


@pytest.mark.parametrize("n", [1, 2, 5, 33, 300])
@pytest.mark.parametrize("form", list(IN_PLACE))
def test_in_place(slots, form, n):
    gen = torch.Generator(device=DEV).manual_seed(n)
    origin = IN_PLACE[form](n, np.random.default_rng(n))
    bufs = [(t, dim) for t, dim in _buffers(gen, n) if n <= 33 or t.numel() < 4e6]
    want = [_want(t, t.clone(), dim, origin) for t, dim in bufs]
    slots.copy_slots([(t, t, dim) for t, dim in bufs], origin)
    for (t, _), w in zip(bufs, want):
        assert torch.equal(t, w)


def test_in_place_at_the_most_slots(slots):
    gen = torch.Generator(device=DEV).manual_seed(1)
    t = torch.randn((2, 1024, 37), device=DEV, generator=gen)
    origin = np.random.default_rng(4).permutation(1024).tolist()
    want = t[:, origin].clone()
    slots.copy_slots([(t, t, 1)], origin)
    assert torch.equal(t, want)
    from burn_dragon_amd.ffi import BdhError

    t = torch.zeros((1025, 4), device=DEV)
    with pytest.raises(BdhError):
        slots.copy_slots([(t, t, 0)], [0] * 1025)


@pytest.mark.parametrize("n,m", [(1, 1), (7, 1), (3, 12), (12, 3), (40, 41)])
def test_to_other_buffers(slots, n, m):
    gen = torch.Generator(device=DEV).manual_seed(n * 100 + m)
    rng = np.random.default_rng(n)
    src, dst = _buffers(gen, m), _buffers(gen, n)
    origin = rng.integers(-2, m, n).tolist()
    kept = [s.clone() for s, _ in src]
    want = [_want(d, s, dim, origin) for (d, dim), (s, _) in zip(dst, src)]
    slots.copy_slots([(d, s, dim) for (d, dim), (s, _) in zip(dst, src)], torch.tensor(origin, dtype=torch.int32, device=DEV))
    for (d, _), w, (s, _), k in zip(dst, want, src, kept):
        assert torch.equal(d, w) and torch.equal(s, k)


@pytest.mark.parametrize("in_place", [True, False])
def test_device_entries_that_name_no_slot_leave_theirs(slots, in_place):
    gen = torch.Generator(device=DEV).manual_seed(3)
    src = torch.randn((6, 50), device=DEV, generator=gen)
    dst = src if in_place else torch.randn((6, 50), device=DEV, generator=gen)
    origin = [5, 6, -3, 2**31 - 1, -2**31, 0]
    want = _want(dst, src.clone(), 0, origin)
    slots.copy_slots([(dst, src, 0)], torch.tensor(origin, dtype=torch.int32, device=DEV))
    assert torch.equal(dst, want)


def test_views_at_odd_places_and_an_empty_buffer(slots):
    raw = torch.arange(4 * 6 + 1, device=DEV, dtype=torch.int8)
    t = raw[1:].reshape(4, 6)  # starts at an odd byte
    want = t[[3, 3, 0, 1]].clone()
    empty = torch.zeros((0, 4, 5), device=DEV)
    slots.copy_slots([(t, t, 0), (empty, empty, 1)], [3, 3, 0, 1])
    assert torch.equal(t, want) and raw[0] == 0


def test_a_captured_map_is_read_at_replay(slots):
    gen = torch.Generator(device=DEV).manual_seed(9)
    t = torch.randn((2, 8, 100), device=DEV, generator=gen)
    origin = torch.arange(8, device=DEV, dtype=torch.int32)
    from burn_dragon_amd import ffi

    ctx = ffi.Context(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots.copy_slots([(t, t, 1)], origin, ctx)
    rng = np.random.default_rng(2)
    for _ in range(5):
        o = rng.integers(-1, 8, 8)
        origin.copy_(torch.from_numpy(o.astype(np.int32)))
        want = _want(t, t.clone(), 1, o.tolist())
        graph.replay()
        assert torch.equal(t, want)


def test_a_buffer_past_four_gib(slots):
    big = torch.empty((5, 900_000_000), device=DEV, dtype=torch.int8)
    for i in range(5):
        big[i].fill_(i + 1)
    slots.copy_slots([(big, big, 0)], [4, 0, -2, -1, 1])
    assert [int(big[i, j]) for i in range(5) for j in (0, 899_999_999)] == [5, 5, 1, 1, 3, 3, 0, 0, 2, 2]
    assert bool((big[0] == 5).all())
