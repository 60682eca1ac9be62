"""Attention of sequences that continue shared prompts (shared_prefix_attention), and the states of their own that they
get (shared_prefix_fork), against the definition in 64 bits, against the sequences' own recurrent states, and under
what serving does with them: calls in a row, graphs, other streams.

Tolerances.  With u = 2^-24 (f32 rounds to nearest), every term q_n rho_nc and (q.k_s) v_sc of an output carries the
roundings of its query and key (the angle and its sine: 8 steps, softplus 4 more; two factors: 24 in all), of its
decay (8), of its products (3) and of the additions it passes through.  One token: at most Nq in the chain of a workgroup's
rows, `parts` and `blocks` <= Nq / 64 + 1 of them, 48 in a block's score, and len for the values.  Many tokens: every sum
in some order of at most Nq, then span.  So |error| <= u * depth * (sum of the terms' magnitudes), depth as written in
`_depth`; the magnitudes come from the same definition with absolute values."""
import numpy as np
import pytest
import torch

from oracle import bdh_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0**-24
ROT = {"rope": orc.ROPE, "alibi": orc.ALIBI, "pope": orc.POPE}


@pytest.fixture(scope="module")
def gpu():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device: the GPU tests must run on the MI355X box")
    from burn_dragon_amd import ffi, recurrent, shared

    return ffi, recurrent, shared


def _turn(x, freqs, pos, rotary):
    """x [...,N] at position pos, in 64 bits (the product of position and frequency is rounded to f32 by definition)."""
    x = x.astype(np.float64)
    if rotary == "alibi":
        return x
    raw = (np.float32(pos) * freqs).astype(np.float32)
    ang = 2 * np.pi * (raw.astype(np.float64) - np.floor(raw.astype(np.float64)))
    if rotary == "pope":
        m = np.log(np.exp(x) + 1)
        return np.concatenate([m * np.cos(ang), m * np.sin(ang)], -1)
    y = np.empty_like(x)
    y[..., 0::2] = x[..., 0::2] * np.cos(ang[0::2]) - x[..., 1::2] * np.sin(ang[0::2])
    y[..., 1::2] = x[..., 1::2] * np.cos(ang[1::2]) + x[..., 0::2] * np.sin(ang[1::2])
    return y


class Case:
    def __init__(self, seed, counts, h, N, d, S, lens, T, rotary, dtype, density=0.3):
        rng = np.random.default_rng(seed)
        self.counts, self.rotary, self.T, self.dtype = list(counts), rotary, T, dtype
        self.B, self.h, self.N, self.d, self.S = sum(counts), h, N, d, S
        self.Nq = 2 * N if rotary == "pope" else N
        self.owner = [g for g, n in enumerate(counts) for _ in range(n)]
        self.lens = np.array([lens[b % len(lens)] for b in range(self.B)], np.int32)
        self.slopes = [2.0 ** (-(i + 1.0)) for i in range(h)] if rotary == "alibi" else None
        self.rate = np.log(np.exp(-np.array(self.slopes, np.float32)).astype(np.float64)) if self.slopes else np.zeros(h)
        from burn_dragon_amd.kernel.linear_attention import build_freqs

        self.freqs = build_freqs(N, 65536.0, ROT[rotary]).numpy().reshape(-1)
        self.start = rng.integers(0, 3000, len(counts))[self.owner]
        rho = torch.from_numpy(rng.standard_normal((len(counts), h, self.Nq, d)).astype(np.float32)).to(dtype)
        self.rho_t, self.rho = rho, rho.to(torch.float64).numpy()

        def act(*shape):
            return (np.maximum(rng.standard_normal(shape) * 2, 0) * (rng.random(shape) < density)).astype(np.float32)

        self.past = act(self.B, h, max(1, int(self.lens.max(initial=0))), N)
        self.x = act(self.B, h, T, N)
        self.v = rng.standard_normal((self.B, T, d)).astype(np.float32)
        self.keys = np.zeros((self.B, h, self.Nq, S), np.float32)
        self.values = np.zeros((self.B, S, d), np.float32)
        for b in range(self.B):
            n = int(self.lens[b])
            self.values[b, :n] = rng.standard_normal((n, d))
            for s in range(n):
                self.keys[b, :, :, s] = _turn(self.past[b, :, s], self.freqs, self.start[b] + s, rotary)

    def device(self, dev=DEV):
        t = {n: torch.from_numpy(getattr(self, n)).to(dev) for n in ("x", "v", "keys", "values", "lens", "freqs")}
        t["rho"] = self.rho_t.to(dev)
        t["positions"] = torch.from_numpy((self.start + self.lens).astype(np.int32)).to(dev)
        return t

    def call(self, shared, t, **more):
        return shared.shared_prefix_attention(t["x"], t["v"], t["rho"], t["keys"], t["values"], t["lens"], t["freqs"],
                                              positions=t["positions"], rotary_embedding=self.rotary,
                                              alibi_slopes=self.slopes, counts=self.counts, **more)

    def exact(self):
        """out, its terms' magnitudes, keys, values"""
        out = np.zeros((self.B, self.h, self.T, self.d))
        mag = np.zeros_like(out)
        keys, values = self.keys.astype(np.float64), self.values.astype(np.float64)
        for b in range(self.B):
            rho = self.rho[self.owner[b]]
            for t in range(self.T):
                k = int(self.lens[b]) + t
                q = _turn(self.x[b, :, t], self.freqs, self.start[b] + k, self.rotary)
                a = np.exp(self.rate * k)[:, None]
                back = np.exp(self.rate[:, None] * (k - np.arange(k)))
                out[b, :, t] = a * np.einsum("hn,hnd->hd", q, rho)
                out[b, :, t] += (np.einsum("hn,hns->hs", q, keys[b, :, :, :k]) * back) @ values[b, :k]
                mag[b, :, t] = a * np.einsum("hn,hnd->hd", np.abs(q), np.abs(rho))
                mag[b, :, t] += (np.einsum("hn,hns->hs", np.abs(q), np.abs(keys[b, :, :, :k])) * back) @ np.abs(values[b, :k])
                keys[b, :, :, k] = q
                values[b, k] = self.v[b, t]
        return out, mag, keys, values


def _depth(c):
    extra = 24 + 8 + 3
    if c.T == 1:
        return extra + c.Nq + 2 * (c.Nq // 64 + 5) + 48 + int(c.lens.max())
    return extra + c.Nq + int(c.lens.max()) + c.T


def _check_read(gpu, c):
    _, _, shared = gpu
    t = c.device()
    out = c.call(shared, t, longest=int(c.lens.max()))
    torch.cuda.synchronize()
    ref, mag, keys, values = c.exact()
    err = np.abs(out.double().cpu().numpy() - ref)
    assert (err <= U * _depth(c) * mag + 1e-37).all(), (err / (mag + 1e-300)).max() / U
    got = t["keys"].double().cpu().numpy()
    new = np.zeros(keys.shape, bool)
    for b in range(c.B):
        new[b, :, :, c.lens[b]:c.lens[b] + c.T] = True
    assert np.array_equal(got[~new], keys[~new])  # what was there stays, the room behind stays zero
    big = np.abs(c.x).max() * 2 + 1
    assert np.abs(got - keys)[new].max(initial=0) <= U * 12 * big
    assert ((got != 0) <= (keys != 0))[new].all()
    assert np.array_equal(t["values"].double().cpu().numpy(), values)
    return out


F32, BF16 = torch.float32, torch.bfloat16
READ = [
    # counts, h, N, d, S, lens, T, rotary, dtype
    ((1,), 1, 2, 4, 4, (0,), 1, "rope", F32),
    ((4,), 4, 256, 256, 32, (3, 21, 0, 31), 1, "alibi", F32),
    ((3, 0, 2), 2, 70, 68, 8, (7, 0, 4), 1, "rope", F32),
    ((2, 1), 3, 33, 12, 12, (5, 11), 1, "alibi", F32),
    ((5,), 2, 31, 132, 16, (9, 15, 0), 1, "pope", F32),
    ((17,), 1, 600, 64, 72, (64, 65, 70, 63), 1, "rope", F32),
    ((16, 1), 2, 514, 128, 8, (2, 7), 1, "rope", BF16),
    ((40,), 1, 130, 192, 4, (1, 3, 0), 1, "rope", F32),
    ((70, 3), 1, 66, 260, 4, (2,), 1, "alibi", BF16),
    ((2,), 1, 300, 1024, 8, (6, 1), 1, "pope", BF16),
    ((2,), 1, 8, 8, 1100, (1060, 1099), 1, "rope", F32),
    ((3,), 5, 1030, 320, 20, (13, 2, 19), 1, "rope", BF16),
    # more blocks of rows than workgroups: several blocks one after the other
    ((20, 3), 16, 16384, 8, 8, (3, 0, 7), 1, "rope", BF16),
    ((18,), 16, 16384, 4, 8, (5, 1), 1, "rope", F32),
    ((40,), 8, 16384, 8, 4, (3, 2), 1, "alibi", F32),
    ((3,), 16, 8192, 12, 8, (7, 2), 1, "pope", BF16),
    ((9, 2), 16, 8192, 16, 16, (3, 5), 7, "rope", BF16),
    ((1,), 1, 2, 4, 4, (0, 2), 2, "rope", F32),
    ((4, 2), 2, 130, 68, 64, (0, 13, 7), 45, "rope", F32),
    ((3, 3), 2, 64, 128, 40, (8, 1), 32, "alibi", F32),
    ((1, 0, 2), 3, 35, 20, 40, (6, 3, 2), 33, "pope", F32),
    ((2, 1), 1, 258, 64, 12, (4, 9), 3, "rope", BF16),
    ((5,), 1, 129, 36, 132, (100, 3), 29, "alibi", BF16),
]


@pytest.mark.parametrize("counts,h,N,d,S,lens,T,rotary,dtype", READ)
def test_attention_equals_the_definition(gpu, counts, h, N, d, S, lens, T, rotary, dtype):
    _check_read(gpu, Case(hash((sum(counts), h, N, d, T)) % 2**31, counts, h, N, d, S, lens, T, rotary, dtype))


@pytest.mark.parametrize("density", [0.0, 1.0])
@pytest.mark.parametrize("T", [1, 6])
def test_silent_and_fully_firing_tokens(gpu, density, T):
    out = _check_read(gpu, Case(7, (3, 2), 2, 200, 64, 24, (0, 11, 18), T, "rope", F32, density))
    if density == 0.0:
        assert not out.any()


def _check_fork(gpu, c, out):
    """u * (len additions + decays 8 + products 3) of the magnitudes; a bf16 state is rounded once more, by half a step."""
    ref = np.zeros((c.B, c.h, c.Nq, c.d))
    mag = np.zeros_like(ref)
    for b in range(c.B):
        n = int(c.lens[b])
        a, back = np.exp(c.rate * n)[:, None, None], np.exp(c.rate[:, None] * (n - np.arange(n)))
        k = c.keys[b, :, :, :n].astype(np.float64) * back[:, None]
        ref[b] = a * c.rho[c.owner[b]] + k @ c.values[b, :n].astype(np.float64)
        mag[b] = a * np.abs(c.rho[c.owner[b]]) + np.abs(k) @ np.abs(c.values[b, :n].astype(np.float64))
    bound = U * (int(c.lens.max()) + 12) * mag
    if c.dtype == BF16:
        bound = bound * (1 + 2.0**-8) + 2.0**-8 * np.abs(ref)
    err = np.abs(out.double().cpu().numpy() - ref)
    assert (err <= bound + 1e-37).all(), (err / (mag + 1e-300)).max() / U


FORK = [
    ((1,), 1, 2, 4, 4, (0,), "rope", F32),
    ((4,), 4, 256, 256, 32, (5, 32, 17), "alibi", F32),
    ((3, 0, 2), 2, 70, 68, 8, (8, 0, 3), "rope", BF16),
    ((2, 1), 3, 33, 12, 12, (5, 11, 12), "alibi", BF16),
    ((2,), 1, 31, 132, 20, (9, 19), "pope", F32),
    ((3,), 1, 260, 1024, 64, (63, 64, 1), "rope", F32),
    ((2,), 2, 9, 64, 1028, (1025, 3), "alibi", F32),
    # several times the rows that a workgroup makes at a time
    ((40, 24), 16, 1000, 8, 12, (7, 12, 0), "rope", F32),
    ((70,), 8, 1010, 8, 72, (71, 64, 0, 33), "alibi", BF16),
    # 65 to 128 tokens, and more, in blocks of 64, 128 and 192 columns
    ((3, 1), 2, 70, 60, 128, (128, 65, 0), "rope", F32),
    ((4, 6), 4, 600, 180, 112, (100, 3, 112, 64), "pope", F32),
    ((9,), 4, 610, 200, 100, (97, 100, 65), "alibi", BF16),
    ((4,), 4, 640, 184, 96, (96, 33), "rope", BF16),
    ((5,), 4, 600, 180, 160, (130, 3, 159), "rope", F32),
]


@pytest.mark.parametrize("counts,h,N,d,S,lens,rotary,dtype", FORK)
def test_fork_equals_the_definition(gpu, counts, h, N, d, S, lens, rotary, dtype):
    _, _, shared = gpu
    c = Case(hash((h, N, d)) % 2**31, counts, h, N, d, S, lens, 1, rotary, dtype)
    t = c.device()
    before = t["rho"].clone()
    out = shared.shared_prefix_fork(t["rho"], t["keys"], t["values"], t["lens"], rotary_embedding=rotary,
                                    alibi_slopes=c.slopes, counts=c.counts)
    _check_fork(gpu, c, out)
    assert torch.equal(before, t["rho"])


@pytest.mark.parametrize("rotary", ["rope", "alibi", "pope"])
def test_steps_equal_those_of_own_states(gpu, rotary):
    """5 tokens at once, then 6 one by one, next to recurrent_attention on a copy of the prompt's state for each sequence:
    both within their bounds of the definition, so of each other within twice the bound of the longer sums."""
    _, recurrent, shared = gpu
    c = Case(11, (3, 2), 2, 96, 64, 16, (0,), 5, rotary, F32)
    t = c.device()
    rho = t["rho"][c.owner].clone()
    rng = np.random.default_rng(3)
    lens, pos = t["lens"], t["positions"]
    scale = 0.0
    for n in [5] + [1] * 6:
        x = torch.from_numpy(np.maximum(rng.standard_normal((5, 2, n, 96)), 0).astype(np.float32)).to(DEV)
        v = torch.from_numpy(rng.standard_normal((5, n, 64)).astype(np.float32)).to(DEV)
        own = recurrent.recurrent_attention(x, v, rho, t["freqs"], 0, rotary_embedding=shared.RotaryEmbedding.parse(rotary),
                                            alibi_slopes=c.slopes, positions=pos)
        out = shared.shared_prefix_attention(x, v, t["rho"], t["keys"], t["values"], lens, t["freqs"], positions=pos,
                                             rotary_embedding=rotary, alibi_slopes=c.slopes, counts=c.counts)
        lens += n
        pos += n
        scale = max(scale, own.abs().max().item())
        assert (out - own).abs().max().item() <= 1e-5 * scale  # u * depth (400) * cancellation (terms over their sum, < 1/2)
    state = shared.shared_prefix_fork(t["rho"], t["keys"], t["values"], lens, rotary_embedding=rotary, alibi_slopes=c.slopes,
                                      counts=c.counts)
    assert (state - rho).abs().max().item() <= 1e-5 * rho.abs().max().item()


@pytest.mark.parametrize("T", [1, 4])
def test_a_sequence_without_room_gets_nan_and_others_their_output(gpu, T):
    _, _, shared = gpu
    c = Case(5, (4,), 2, 40, 64, 16, (3, 8, 5, 2), T, "rope", F32)
    t = c.device()
    good = c.call(shared, t)
    t = c.device()
    t["lens"][1] = 17
    t["lens"][2] = -1
    keys, values = t["keys"].clone(), t["values"].clone()
    out = c.call(shared, t)
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all()
    assert torch.equal(out[0], good[0]) and torch.equal(out[3], good[3])
    assert torch.equal(t["keys"][1:3], keys[1:3]) and torch.equal(t["values"][1:3], values[1:3])
    state = shared.shared_prefix_fork(t["rho"], t["keys"], t["values"], t["lens"], counts=c.counts)
    assert torch.isnan(state[1]).all() and torch.isnan(state[2]).all() and torch.isfinite(state[[0, 3]]).all()


def test_equal_calls_give_equal_bits(gpu):
    _, _, shared = gpu
    for T in (1, 7):
        c = Case(9, (33, 4), 2, 300, 128, 24, (13, 2), T, "rope", F32)
        outs = []
        for _ in range(3):
            t = c.device()
            outs.append((c.call(shared, t), t["keys"]))
        assert all(torch.equal(o, outs[0][0]) and torch.equal(k, outs[0][1]) for o, k in outs)


def test_graph_replays_walk_on(gpu):
    """A step and the advance of lens and positions in one graph: every replay is the next token, checked against eager
    steps, with eager work of another shape between the replays."""
    ffi, _, shared = gpu
    c = Case(21, (6,), 2, 128, 64, 16, (2, 5), 1, "rope", F32)
    other = Case(22, (2,), 1, 64, 32, 8, (1,), 3, "alibi", F32)
    ctx = ffi.Context(0)
    rng = np.random.default_rng(8)
    xs = torch.from_numpy(np.maximum(rng.standard_normal((7, 6, 2, 1, 128)), 0).astype(np.float32)).to(DEV)
    vs = torch.from_numpy(rng.standard_normal((7, 6, 1, 64)).astype(np.float32)).to(DEV)

    def step(t, x, v):
        o = shared.shared_prefix_attention(x, v, t["rho"], t["keys"], t["values"], t["lens"], t["freqs"],
                                           positions=t["positions"], counts=c.counts, ctx=ctx)
        for p in ("lens", "positions"):
            ctx.check(ctx.lib.bdh_advance_positions(ctx.handle, t[p].data_ptr(), 6, 1))
        return o

    t = c.device()
    want = [step(t, x, v).clone() for x, v in zip(xs, vs)]
    end = t["keys"].clone()
    t = c.device()
    x, v = xs[0].clone(), vs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = step(t, x, v)
    for i in range(7):
        x.copy_(xs[i])
        v.copy_(vs[i])
        graph.replay()
        assert torch.equal(out, want[i]), i
        o = other.device()
        other.call(shared, o)
        torch.cuda.synchronize()
    assert torch.equal(t["keys"], end)


def test_another_stream_and_two_contexts(gpu):
    ffi, _, shared = gpu
    c = Case(31, (8,), 2, 128, 64, 16, (2, 5), 1, "rope", F32)
    t = c.device()
    want = c.call(shared, t)
    torch.cuda.synchronize()
    a, b = ffi.Context(0), ffi.Context(0)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    ta, tb = c.device(), c.device()
    torch.cuda.synchronize()
    with torch.cuda.stream(sa):
        oa = c.call(shared, ta, ctx=a)
    with torch.cuda.stream(sb):
        ob = c.call(shared, tb, ctx=b)
    torch.cuda.synchronize()
    assert torch.equal(oa, want) and torch.equal(ob, want)


# more than 32 tokens of a prompt's sequences: dense products, their sums dealt to several workgroups, even and uneven prompts;
# a large bf16 state, and prompts most of which have few, take tiles of 32
DENSE = [
    ((2,), 16, 16384, 68, 24, (3, 0), 18, "rope", BF16),
    ((20, 1, 1), 1, 512, 64, 8, (3, 0), 3, "rope", F32),
    ((9, 30), 2, 1025, 72, 8, (3, 0, 4), 1, "pope", BF16),
    ((9, 65), 2, 1024, 72, 24, (3, 20, 17), 1, "rope", F32),
    ((33,), 4, 256, 256, 32, (16, 20, 15, 31), 1, "alibi", F32),
    ((2, 2), 2, 8192, 64, 32, (3, 9, 0), 20, "rope", F32),
    ((3, 0, 1), 2, 8190, 72, 24, (5, 1), 14, "rope", F32),
    ((1, 4), 1, 5001, 36, 48, (7, 0, 11), 35, "pope", BF16),
    ((7,), 3, 2048, 128, 12, (2, 4, 0), 5, "alibi", BF16),
    ((17,), 1, 4000, 64, 4, (1, 2), 2, "rope", F32),
    ((5, 28), 2, 512, 256, 8, (0, 5, 3), 3, "alibi", F32),
    ((2,), 1, 300, 64, 132, (0,), 129, "rope", F32),
    ((2, 5), 2, 8192, 64, 32, (3, 8, 0), 24, "rope", F32),
    ((1, 0, 6), 2, 4101, 68, 48, (3, 18, 0), 30, "pope", BF16),
    ((3, 3), 4, 2047, 128, 16, (6, 0), 10, "alibi", BF16),
]


@pytest.mark.parametrize("counts,h,N,d,S,lens,T,rotary,dtype", DENSE)
def test_many_tokens_equal_the_definition(gpu, counts, h, N, d, S, lens, T, rotary, dtype):
    _check_read(gpu, Case(hash((sum(counts), h, N, d, T)) % 2**31, counts, h, N, d, S, lens, T, rotary, dtype, 0.1))


@pytest.mark.parametrize("counts,N,T", [((20, 3), 700, 2), ((20, 3), 700, 7), ((11, 11), 4096, 7), ((20, 3), 8192, 7)])
def test_a_sequence_without_room_among_many_tokens(gpu, counts, N, T):
    _, _, shared = gpu
    c = Case(6, counts, 2, N, 64, 16, (3, 8, 5, 2), T, "rope", F32)
    t = c.device()
    good = c.call(shared, t)
    t = c.device()
    t["lens"][1], t["lens"][21] = 17, -1
    keys, values = t["keys"].clone(), t["values"].clone()
    out = c.call(shared, t)
    bad = [1, 21]
    rest = [b for b in range(c.B) if b not in bad]
    assert torch.isnan(out[bad]).all() and torch.equal(out[rest], good[rest])
    assert torch.equal(t["keys"][bad], keys[bad]) and torch.equal(t["values"][bad], values[bad])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_fork_does_not_look_behind_the_last_token(gpu, dtype):
    _, _, shared = gpu
    c = Case(41, (4,), 2, 70, 68, 72, (5, 0, 66, 31), 1, "rope", dtype)
    t = c.device()
    for b in range(4):
        t["keys"][b, :, :, c.lens[b]:] = float("nan")
        t["values"][b, c.lens[b]:] = float("inf")
    _check_fork(gpu, c, shared.shared_prefix_fork(t["rho"], t["keys"], t["values"], t["lens"], counts=c.counts))


def test_two_graphs_of_one_workspace(gpu):
    """Steps of two shapes captured on one context, replayed in turns with eager calls of a third between them: each leaves
    what its eager call leaves."""
    ffi, _, shared = gpu
    cases = [Case(51, (9,), 2, 256, 64, 16, (2, 5), 1, "rope", F32), Case(52, (3, 2), 2, 130, 128, 24, (4, 9), 12, "alibi", BF16)]
    between = Case(53, (2, 4), 1, 64, 32, 8, (1,), 3, "pope", F32)
    ctx = ffi.Context(0)
    want, held, graphs = [], [], []
    for c in cases + [between]:
        t = c.device()
        want.append((c.call(shared, t, ctx=ctx), t["keys"]))
    torch.cuda.synchronize()
    for c in cases:
        t = c.device()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c.call(shared, t, ctx=ctx)
        held.append((t, out))
        graphs.append(graph)
    for i in range(6):
        k = i % 2
        held[k][1].fill_(-1.0)
        graphs[k].replay()
        assert torch.equal(held[k][1], want[k][0]) and torch.equal(held[k][0]["keys"], want[k][1]), i
        t = between.device()
        assert torch.equal(between.call(shared, t, ctx=ctx), want[2][0])


# rows of four numbers; 17 to 32 tokens of a prompt's sequences, alone and next to prompts of few
FORMS = [
    ((2,), 1, 6, 4, 8, (1, 3), 1, "rope", BF16),
    ((20,), 2, 130, 4, 4, (1, 0), 1, "alibi", BF16),
    ((5,), 1, 33, 4, 12, (2, 7), 5, "pope", BF16),
    ((3,), 1, 10, 4, 8, (2, 0), 3, "rope", BF16),
    ((4,), 2, 300, 64, 16, (3, 0), 7, "rope", F32),
    ((10, 1, 1), 2, 513, 100, 12, (3, 0, 6), 2, "alibi", F32),
    ((22, 2, 3), 1, 1030, 72, 8, (3, 0, 6), 1, "rope", F32),
    ((10, 1), 2, 140, 136, 12, (3, 0, 6), 3, "pope", BF16),
]


@pytest.mark.parametrize("counts,h,N,d,S,lens,T,rotary,dtype", FORMS)
def test_every_form_equals_the_definition(gpu, counts, h, N, d, S, lens, T, rotary, dtype):
    _check_read(gpu, Case(hash((sum(counts), h, N, d, T)) % 2**31, counts, h, N, d, S, lens, T, rotary, dtype))


@pytest.mark.parametrize("T", [1, 20])
def test_caches_beyond_32_bits_of_places(gpu, T):
    """Three sequences of 2 heads of 8192 neurons with room for 131072 tokens: 26 GB of keys.  The last sequence is nearly full;
    its last head, and the fork of it, against the definition in 64 bits."""
    _, _, shared = gpu
    B, h, N, d, S = 3, 2, 8192, 64, 131072
    n = S - T - 1
    gen = torch.Generator(DEV).manual_seed(5)
    rand = lambda *shape: torch.randn(shape, device=DEV, generator=gen)
    keys = torch.zeros((B, h, N, S), device=DEV)
    keys[2, 1, :, :n] = rand(N, n)
    values = torch.zeros((B, S, d), device=DEV)
    values[2, :n] = rand(n, d)
    lens = torch.tensor([0, 3, n], dtype=torch.int32, device=DEV)
    x = rand(B, h, T, N).relu() * (torch.rand((B, h, T, N), device=DEV, generator=gen) < 0.05)
    v, rho = rand(B, T, d), rand(1, h, N, d)
    state = shared.shared_prefix_fork(rho, keys, values, lens, rotary_embedding="alibi", alibi_slopes=[1e-5, 1e-5])
    out = shared.shared_prefix_attention(x, v, rho, keys, values, lens, None, rotary_embedding="alibi", alibi_slopes=[1e-5, 1e-5])
    rate = float(np.log(np.exp(-np.float32(1e-5)).astype(np.float64)))
    q, K, V = x[2, 1].double(), keys[2, 1, :, :n + T], values[2, :n + T].double()
    scores = torch.zeros((T, n + T), dtype=torch.float64, device=DEV)
    size = torch.zeros_like(scores)
    ref, mag = torch.zeros((N, d), dtype=torch.float64, device=DEV), torch.zeros((N, d), dtype=torch.float64, device=DEV)
    back = torch.exp(rate * (n - torch.arange(n, device=DEV, dtype=torch.float64)))[:, None]
    for a in range(0, N, 1024):
        part = K[a:a + 1024].double()
        scores += q[:, a:a + 1024] @ part
        size += q[:, a:a + 1024].abs() @ part.abs()
        ref[a:a + 1024] = part[:, :n] @ (V[:n] * back)
        mag[a:a + 1024] = part[:, :n].abs() @ (V[:n] * back).abs()
    k = n + torch.arange(T, device=DEV)[:, None]
    decay = torch.exp(rate * (k - torch.arange(n + T, device=DEV)).double()) * (torch.arange(n + T, device=DEV) < k)
    grown = torch.exp(rate * k.double())
    want = grown * (q @ rho[0, 1].double()) + (scores * decay) @ V
    terms = grown * (q.abs() @ rho[0, 1].double().abs()) + (size * decay) @ V.abs()
    depth = 35 + N + 2 * (N // 64 + 5) + 48 + n + T
    assert ((out[2, 1].double() - want).abs() <= U * depth * terms).all()
    assert torch.equal(keys[2, 1, :, n:n + T], x[2, 1].t()) and torch.equal(values[2, n:n + T], v[2])
    assert not keys[2, 1, :, n + T:].any() and not keys[1, 1, :, 3 + T:].any()
    start = float(np.exp(rate * n)) * rho[0, 1].double()
    assert ((state[2, 1].double() - ref - start).abs() <= U * (n + 12) * (mag + start.abs())).all()
    assert torch.equal(state[0], rho[0])


@pytest.mark.parametrize("counts,h,N", [((4, 2), 2, 514), ((3, 3), 4, 4096), ((4, 2), 4, 8192)])
def test_captured_forks_and_reads_of_many_tokens(gpu, counts, h, N):
    """Many tokens, then the fork of what they left, in one graph: replays on other inputs equal eager calls, with eager work
    between them."""
    ffi, _, shared = gpu
    ctx = ffi.Context(0)
    c = Case(61, counts, h, N, 64, 32, (3, 0, 9), 14, "rope", F32)

    def run(t, x):
        out = shared.shared_prefix_attention(x, t["v"], t["rho"], t["keys"], t["values"], t["lens"], t["freqs"],
                                             positions=t["positions"], counts=c.counts, ctx=ctx)
        return out, shared.shared_prefix_fork(t["rho"], t["keys"], t["values"], t["lens"] + 14, counts=c.counts, ctx=ctx)

    xs = [c.device()["x"] * (1 + 0.25 * i) for i in range(4)]
    want = [run(c.device(), x) for x in xs]
    t, x = c.device(), xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, state = run(t, x)
    for i in (0, 1, 2, 3, 1, 0):
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(out, want[i][0]) and torch.equal(state, want[i][1]), i
        again = run(c.device(), xs[3])
        torch.cuda.synchronize()
        assert torch.equal(again[0], want[3][0])


@pytest.mark.parametrize("counts,h,N,d,S,lens,T,rotary,dtype", [
    ((1,), 1, 64, 16, 1004, (3,), 1000, "rope", F32), ((1,), 1, 512, 128, 1004, (3,), 1000, "alibi", F32),
    ((1,) * 256, 1, 34, 12, 8, (3, 0, 5), 1, "rope", BF16), ((1, 0) * 128, 2, 20, 8, 12, (3, 0, 5), 4, "pope", F32),
    ((9,), 64, 16, 4, 8, (2, 5), 1, "alibi", F32), ((2, 1), 64, 18, 8, 8, (2, 5), 3, "alibi", BF16)])
def test_long_calls_many_prompts_and_many_heads(gpu, counts, h, N, d, S, lens, T, rotary, dtype):
    _check_read(gpu, Case(77, counts, h, N, d, S, lens, T, rotary, dtype))


@pytest.mark.parametrize("T", [1, 3])
def test_as_many_sequences_as_a_call_takes(gpu, T):
    """65535 sequences alike: each within the bound of the definition."""
    _, _, shared = gpu
    one, B = Case(78, (1,), 1, 20, 8, 8, (3,), T, "rope", F32), 65535
    t = one.device()
    many = {n: t[n][:1].expand(B, *t[n].shape[1:]).contiguous() for n in ("x", "v", "keys", "values", "lens", "positions")}
    many.update(rho=t["rho"], freqs=t["freqs"])
    ref, mag, keys, _ = one.exact()
    one.counts = [B]
    got = one.call(shared, many)
    bound = torch.from_numpy(U * _depth(one) * mag[:1]).to(DEV)
    assert ((got.double() - torch.from_numpy(ref[:1]).to(DEV)).abs() <= bound).all()
    assert torch.equal(many["keys"], many["keys"][:1].expand_as(many["keys"]))
    assert np.array_equal(many["keys"][0].cpu().numpy() != 0, keys[0] != 0)
    state = shared.shared_prefix_fork(t["rho"], many["keys"], many["values"], many["lens"] + T, counts=[B])
    assert torch.equal(state, state[:1].expand_as(state)) and torch.isfinite(state[0]).all()


def test_many_tokens_without_room_for_dense_products(gpu):
    """A context whose workspace may not hold the state in f32 makes the call as it makes one of few tokens, and refuses what
    it has no room for at all."""
    ffi, _, shared = gpu
    c = Case(91, (3, 3), 4, 2047, 128, 16, (6, 0), 10, "alibi", BF16)
    ref, mag, keys, _ = c.exact()
    for mib in (0, 7):
        ctx = ffi.Context(0)
        ctx.set_option("workspace.max_mib", mib)
        t = c.device()
        out = c.call(shared, t, ctx=ctx)
        assert (np.abs(out.double().cpu().numpy() - ref) <= U * _depth(c) * mag).all()
        assert np.array_equal(t["keys"].double().cpu().numpy(), keys)
    ctx.close()
    ctx = ffi.Context(0)
    ctx.set_option("workspace.max_mib", 1)
    with pytest.raises(ffi.BdhError, match="workspace"):
        c.call(shared, c.device(), ctx=ctx)
    ctx.close()


# sequences, tokens, columns, state: the f32 cores, split f32 states, bf16 states, several tokens of few
@pytest.mark.parametrize("B,T,d,dtype", [(4, 1, 64, F32), (20, 1, 64, F32), (4, 1, 64, BF16), (20, 1, 132, BF16), (3, 9, 64, F32),
                                         (2, 3, 64, BF16)])
def test_the_largest_numbers_of_f32(gpu, B, T, d, dtype):
    """Numbers between the largest of bf16 (3.3895e38) and the largest of f32, in the prompt's state (f32) or among the activations:
    sums that f32 holds are what the definition gives, to the bound of one product (24 + 8 + 3 roundings and one term)."""
    _, _, shared = gpu
    rng = np.random.default_rng(13)
    N, h, top = 130, 2, float(np.finfo(np.float32).max)
    many = np.float32(top) * np.float32(1) - np.float32(2.0**104) * rng.integers(0, 2**15, (h, N, d)).astype(np.float32)
    assert (many > 3.3895e38).all() and np.isfinite(many).all()
    small = (rng.integers(1, 4, (h, N, d)) / 8).astype(np.float32)
    for large_state in ([True, False] if dtype == F32 else [False]):
        x = np.zeros((B, h, T, N), np.float32)
        for b in range(B):
            for i in range(h):
                x[b, i, np.arange(T), rng.choice(N, T, replace=False)] = 0.25 if large_state else many[i, 0, 0]
        rho = torch.from_numpy(many if large_state else small).to(dtype)[None]
        keys, values = torch.zeros((B, h, N, 12), device=DEV), torch.zeros((B, 12, d), device=DEV)
        lens = torch.zeros(B, dtype=torch.int32, device=DEV)
        out = shared.shared_prefix_attention(torch.from_numpy(x).to(DEV), torch.zeros((B, T, d), device=DEV), rho.to(DEV), keys, values,
                                             lens, None, rotary_embedding="alibi", alibi_slopes=[0.0] * h)
        want = np.einsum("bhtn,hnd->bhtd", x.astype(np.float64), rho[0].double().numpy())
        assert (np.abs(out.double().cpu().numpy() - want) <= U * 36 * want).all()
        assert torch.equal(keys[:, :, :, :T].permute(0, 1, 3, 2).cpu(), torch.from_numpy(x))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_largest_numbers_of_f32_in_a_fork(gpu, dtype):
    """As above, in keys and in values; a token of keys 0 is of no use to the others."""
    _, _, shared = gpu
    N, d, S = 34, 68, 8
    top = np.float32(np.finfo(np.float32).max)
    keys, values = np.zeros((2, 1, N, S), np.float32), np.zeros((2, S, d), np.float32)
    keys[0, 0, :17, 2], values[0, 2] = 0.25, top  # values, and further down keys
    keys[0, 0, 17:, 5], values[0, 5] = -top, 0.125
    keys[1, 0, 5, 0], values[1, 0] = -top, -0.25
    rho = torch.ones((1, 1, N, d), device=DEV, dtype=dtype)
    lens = torch.tensor([8, 3], dtype=torch.int32, device=DEV)
    out = shared.shared_prefix_fork(rho, torch.from_numpy(keys).to(DEV), torch.from_numpy(values).to(DEV), lens)
    want = 1 + np.einsum("bhns,bsd->bhnd", keys.astype(np.float64), values.astype(np.float64))
    bound = U * 20 * np.abs(want)
    if dtype == BF16:
        bound = bound * (1 + 2.0**-8) + 2.0**-8 * np.abs(want)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("counts,h,N,d,S,T", [((32,), 4, 256, 64, 2048, 1), ((20, 1, 3), 2, 512, 128, 2048, 1), ((2,), 4, 256, 64, 4096, 8),
                                              ((3,), 2, 1030, 512, 2048, 5), ((3,), 4, 1024, 256, 2048, 20), ((1, 4), 4, 2048, 128, 1024, 30)])
def test_the_workspace_does_not_grow_with_the_answers(gpu, counts, h, N, d, S, T):
    """Calls of one shape on a context of their own, longest from 0 to what the capacity takes: after the first one the workspace
    may not grow any more (a limit of 1 MiB refuses every growth), and what comes out is what a context without a past gives."""
    ffi, _, shared = gpu
    B = sum(counts)
    gen = torch.Generator(DEV).manual_seed(6)
    x = torch.randn((B, h, T, N), device=DEV, generator=gen).relu() * (torch.rand((B, h, T, N), device=DEV, generator=gen) < 0.05)
    v, rho = torch.randn((B, T, d), device=DEV, generator=gen), torch.randn((len(counts), h, N, d), device=DEV, generator=gen)
    keys, values = torch.zeros((B, h, N, S), device=DEV), torch.zeros((B, S, d), device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)

    def call(ctx, longest):
        return shared.shared_prefix_attention(x, v, rho, keys, values, lens, None, rotary_embedding="alibi", alibi_slopes=[0.1] * h,
                                              counts=counts, longest=longest, ctx=ctx)

    walker = ffi.Context(0)
    call(walker, 0)
    walker.set_option("workspace.max_mib", 1)
    for longest in (0, 1, 60, 64, 200, S // 3, S // 2 + 1, S - T):
        got = call(walker, longest)
        fresh = ffi.Context(0)
        assert torch.equal(got, call(fresh, longest)), longest
        torch.cuda.synchronize()
        fresh.close()
    call(walker, None)
    torch.cuda.synchronize()
    walker.close()
