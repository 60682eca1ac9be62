"""Packed products called from graphs, streams and contexts.

This file runs last: streams share a few hardware queues in the order in which they are first used, and the tests of contexts with
a stream of their own, which hold one stream while another goes on, need the two on different queues."""
import pytest
import torch

from .test_gpu_packed import BF16, DEV, F32, INT8, close, definition, gen, pack, rows_of

pytestmark = pytest.mark.gpu


def _calls(kind, seed=0):
    """One call of each way a product is made: streamed rows, parts of a long k, tiles, tiles of parts, groups, gates."""
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import grouped_product, product

    g = gen(seed)
    r = lambda *shape: torch.randn(shape, generator=g).to(DEV)
    calls = []
    for M, K, N in ((3, 256, 200), (20, 9000, 70), (300, 256, 300), (130, 5000, 64), (70, 64, 64)):
        w, x = pack(r(K, N).cpu(), kind), r(M, K)
        calls.append(([x], lambda x, w=w: product(x, w)))
    w3 = pack(r(3, 96, 80).cpu(), kind)
    for M in (20, 200):
        offsets = torch.tensor([0, M // 4, M // 4, M], dtype=torch.int32, device=DEV)
        calls.append(([r(M, 96), offsets], lambda x, o: grouped_product(x, w3, o)))
    for T in (1, 90):
        calls.append(([r(2, 3, T, 96), r(2, 3, T, 80)], lambda x, m: packed_forward(x, w3, gate=m)))
    return calls


@pytest.mark.parametrize("kind", [INT8, BF16])
def test_graphs_share_no_workspace(kind):
    """Every call captured in a graph of its own, all of them kept; replayed in turn with new inputs, eager calls of larger
    shapes in between."""
    calls = _calls(kind)
    graphs = []
    for inputs, call in calls:
        call(*inputs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(*inputs)
        graphs.append((graph, out))
    for turn in range(4):
        for (inputs, call), (graph, out) in zip(calls, graphs):
            inputs[0].copy_(torch.randn(inputs[0].shape, generator=gen(turn)))
            graph.replay()
        torch.cuda.synchronize()
        for inputs, call in _calls(kind, 100 + turn):
            call(*inputs)
        for k, ((inputs, call), (graph, out)) in enumerate(zip(calls, graphs)):
            assert torch.equal(call(*inputs), out), (turn, k)


@pytest.mark.parametrize("kind", [INT8, BF16])
def test_two_streams_at_once(kind):
    from burn_dragon_amd import ffi
    from burn_dragon_amd.packed import product

    g = gen(5)
    w = pack(torch.randn((700, 300), generator=g), kind)
    xs = [torch.randn((400, 700), generator=g).to(DEV) for _ in range(2)]
    want = [product(x, w).clone() for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    contexts = []
    for s in streams:
        with torch.cuda.stream(s):
            contexts.append(ffi.Context(0, s.cuda_stream))
    got = [[], []]
    for _ in range(20):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(product(xs[k], w, ctx=contexts[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, want[k]) for o in got[k])


def test_a_context_that_keeps_its_stream():
    """What the wrapper makes (results, workspaces, copies of rows that are none) is made on the context's stream."""
    from burn_dragon_amd import ffi
    from burn_dragon_amd.packed import grouped_product, product

    g = gen(6)
    w, w2 = pack(torch.randn((100, 90), generator=g), INT8), pack(torch.randn((2, 100, 90), generator=g), INT8)
    x = torch.randn((100, 150), generator=g).to(DEV).t()  # columns first: copied to rows
    rows = x.contiguous()
    want, want2 = product(x, w), grouped_product(rows, w2, [0, 70, 150])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    ctx = ffi.Context(0, side.cuda_stream)
    for _ in range(10):
        got, got2 = product(x, w, ctx=ctx), grouped_product(rows, w2, [0, 70, 150], ctx=ctx)
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(got2, want2)


def test_results_do_not_depend_on_the_company_of_a_row():
    """8 bits: a row's result is the same alone, among few, among many, in a group and as one of several heads' rows."""
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import grouped_product, product

    g = gen(7)
    w = torch.randn((300, 200), generator=g)
    packed, x = pack(w, INT8), torch.randn((500, 300), generator=g).to(DEV)
    many = product(x, packed)
    assert torch.equal(product(x[:40], packed), many[:40]) and torch.equal(product(x[7:8], packed), many[7:8])
    both = pack(torch.stack([w, w.flip(1)]), INT8)
    assert torch.equal(grouped_product(x, both, [0, 210, 500])[:210], many[:210])
    assert torch.equal(grouped_product(x[:30], both, [0, 21, 30])[:21], many[:21])
    heads = packed_forward(x.reshape(1, 1, 500, 300), both)
    assert torch.equal(heads[0, 0], many.clamp(min=0)) and torch.equal(heads[0, 1], many.clamp(min=0).flip(1))


def test_calls_are_repeatable():
    for kind in (INT8, BF16):
        for inputs, call in _calls(kind):
            first = call(*inputs).clone()
            for _ in range(3):
                assert torch.equal(call(*inputs), first)


def test_the_c_entry_refuses_a_workspace_that_is_too_small():
    from burn_dragon_amd import ffi

    ctx = ffi.context_on(0)
    w = pack(torch.ones(64, 64), INT8)
    size = lambda n: ctx.lib.bdh_packed_workspace(ctx.handle, w._ref, n, n, None, ffi.F32, 64)
    M = next(n for n in (100, 10000, 1000000) if size(n) > 0)  # few rows need none
    x, out, need = torch.zeros(M, 64, device=DEV), torch.full((M, 64), 7.0, device=DEV), size(M)
    ws = torch.empty(need + 16, dtype=torch.uint8, device=DEV)
    run = lambda p, n, o=out: ctx.lib.bdh_packed_product(ctx.handle, w._ref, M, x.data_ptr(), ffi.F32, 64, o.data_ptr(), ffi.F32, 64, p, n)
    assert run(None, 0) == ffi.E_INVAL and run(ws.data_ptr(), need - 1) == ffi.E_INVAL and run(ws.data_ptr() + 4, need) == ffi.E_ALIGN
    assert run(x.data_ptr(), need) == ffi.E_INVAL and run(ws.data_ptr(), need, x) == ffi.E_INVAL
    assert (out == 7).all()
    assert run(ws.data_ptr(), need) == ffi.OK and (out == 0).all()


@pytest.mark.parametrize("G", [1, 2, 8, 40])
@pytest.mark.parametrize("M", [1, 16, 17, 32, 33, 48, 64, 65])
def test_few_rows_of_wide_groups(M, G):
    """Whatever a call needs beside its arguments it asks for, on both sides of every rule for few rows."""
    from burn_dragon_amd.packed import grouped_product, product

    K, N = 64, 1500 if G > 1 else 20000
    g = gen(M + G)
    x, w = rows_of(g, M, K, F32), torch.randn((G, K, N), generator=g)
    for kind in (INT8, BF16):
        limits = [i * M // G for i in range(G + 1)]
        got = grouped_product(x.to(DEV), pack(w, kind), limits)
        for k in range(G):
            a, b = limits[k], limits[k + 1]
            if b > a:
                close(got[a:b], *definition(x[a:b], w[k], kind), k)
        if G == 1:
            close(product(x.to(DEV), pack(w, kind)), *definition(x, w[0], kind))


def _room(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"{gib} GiB of memory")


def test_results_beyond_2_31_values():
    """Rows repeat every 40 and 8-bit results do not depend on their neighbours: every block of 40 is the first one's."""
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import product

    _room(24)
    g = gen(5)
    M, K, N = 40000, 64, 65536
    x, w = rows_of(g, 40, K, BF16), torch.randn((K, N), generator=g)
    packed = pack(w, INT8)
    out = product(x.to(DEV, BF16).repeat(M // 40, 1), packed, out_dtype=BF16)
    assert out.numel() > 2**31
    want, bound = definition(x, w, INT8)
    close(out[:40], want, bound + 2.0**-8 * (abs(want) + bound))
    assert all(torch.equal(out[i:i + 4000].view(-1, 40, N), out[:40].expand(100, 40, N)) for i in range(0, M, 4000))
    del out
    w4 = pack(w.view(K, 4, N // 4).transpose(0, 1).contiguous(), INT8)
    gate = torch.randn((1, 4, 40, N // 4), generator=g).to(DEV, BF16)
    out = packed_forward(x.to(DEV, BF16).repeat(M // 40, 1).view(1, 1, M, K), w4, gate=gate.repeat(1, 1, M // 40, 1), out_dtype=BF16)
    first = packed_forward(x.to(DEV, BF16).view(1, 1, 40, K), w4, gate=gate, out_dtype=BF16)
    assert torch.equal(out[:, :, :40], first)
    for h in range(4):
        assert all(torch.equal(out[0, h, i:i + 4000].view(-1, 40, N // 4), first[0, h].expand(100, 40, N // 4)) for i in range(0, M, 4000))


def test_rows_beyond_2_31_values():
    from burn_dragon_amd.packed import product

    _room(16)
    g = gen(6)
    M, K, N = 16800, 131072, 40
    x, w = rows_of(g, 40, K, BF16), torch.randn((K, N), generator=g)
    out = product(x.to(DEV, BF16).repeat(M // 40, 1), pack(w, INT8))
    close(out[:40], *definition(x, w, INT8))
    assert torch.equal(out.view(-1, 40, N), out[:40].expand(M // 40, 40, N))


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("M", [3, 90])
def test_weights_beyond_2_31_bytes(M, kind):
    from burn_dragon_amd.packed import PackedWeights, product

    _room(24)
    g = gen(7)
    K, N = 8192, 64 * 4200
    x, w = rows_of(g, M, K, F32), torch.randn((K, 64), generator=g)
    packed = PackedWeights(w.to(DEV, BF16).repeat(1, N // 64), dtype=kind)
    assert packed.data.numel() > 2**31
    out = product(x.to(DEV), packed)
    close(out[:, -64:], *definition(x, w.to(BF16).float(), kind))
    assert torch.equal(out.view(M, -1, 64), out[:, None, :64].expand(M, N // 64, 64))
