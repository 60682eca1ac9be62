"""Models whose projections are packed: against the same model in 64 bits, and the operators of a layer one after the other."""
import dataclasses

import numpy as np
import pytest
import torch

from oracle import bdh_oracle as orc

from .packed_reference import forward_with_state
from .test_gpu_packed import BF16, DEV, F32, INT8, close, definition, gen

pytestmark = pytest.mark.gpu


def build(shape, weights, **kw):
    from burn_dragon_amd import BDH, BDHConfig, FusedKernelConfig, RotaryEmbedding

    config = BDHConfig(n_layer=shape.n_layer, n_embd=shape.n_embd, n_head=shape.n_head,
                       mlp_internal_dim_multiplier=shape.mlp_internal_dim_multiplier, vocab_size=shape.vocab_size,
                       fused_kernels=FusedKernelConfig(rotary_embedding=RotaryEmbedding(shape.rotary), relu_threshold=shape.relu_threshold))
    names = [f.name for f in dataclasses.fields(weights)]
    return BDH(config, DEV, weights={n: np.asarray(getattr(weights, n), np.float32) for n in names}, **kw)


# Seeds for which no value of a row lies within 2e-3 steps of a border between two whole numbers (or two bf16 numbers): a relative
# error of 1.6e-5 in 8 bits, 8e-6 in bf16, would move none of them to the other side, and f32 roundings stay below.  The logits then
# differ by roundings alone: some twenty in a row behind another, each amplified less than ten times by a LayerNorm: 1e-4.
@pytest.mark.parametrize("rotary,kind,size,seed", [
    (orc.ALIBI, INT8, (2, 32, 2, 4, 2, 3), 115), (orc.ROPE, INT8, (2, 32, 2, 4, 2, 3), 82), (orc.POPE, INT8, (1, 24, 3, 4, 2, 3), 8),
    (orc.ROPE, BF16, (2, 32, 2, 4, 2, 3), 54), (orc.ALIBI, BF16, (2, 32, 2, 4, 2, 3), 139)])
def test_logits_and_state(rotary, kind, size, seed):
    L, d, h, mult, B, T = size
    shape = orc.BDHShape(n_layer=L, n_embd=d, n_head=h, mlp_internal_dim_multiplier=mult, vocab_size=11, rotary=rotary)
    w = orc.init_weights(shape, seed)
    wide = orc.BDHWeights(**{f.name: getattr(w, f.name).astype(np.float64) for f in dataclasses.fields(w)})
    rng = np.random.default_rng(seed)
    tokens, following = rng.integers(0, 11, (B, T)), rng.integers(0, 11, (B, 1))
    state, near = orc.ModelState(L), []
    want = [forward_with_state(shape, wide, t, state, kind, near) for t in (tokens, following)]
    assert min(near) > 2e-3
    model = build(shape, w)
    plain = model.forward_with_state(torch.from_numpy(tokens), model.init_state())
    model.pack_projections(kind)
    mine = model.init_state()
    for t, logits in zip((tokens, following), want):
        got = model.forward_with_state(torch.from_numpy(t), mine).double().cpu().numpy()
        assert np.abs(got - logits).max() <= 1e-4 * np.abs(logits).max()
    for layer in range(L):
        rho = state.rho[layer]
        assert np.abs(mine.storage[layer].double().cpu().numpy() - rho).max() <= 1e-4 * np.abs(rho).max()
    model.pack_projections(None)
    assert torch.equal(model.forward_with_state(torch.from_numpy(tokens), model.init_state()), plain)


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("B,T,h,N,d,rotary", [(2, 1, 4, 256, 256, "alibi"), (3, 40, 2, 130, 64, "rope"), (20, 1, 2, 512, 128, "rope"),
                                              (1, 150, 4, 256, 256, "rope")])
def test_the_operators_of_a_layer(B, T, h, N, d, rotary, kind):
    """D_x, the state step, D_y with its gate and E, each on what the one before left."""
    from burn_dragon_amd import RotaryEmbedding
    from burn_dragon_amd.kernel.linear_attention import build_freqs
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import PackedWeights, product
    from burn_dragon_amd.recurrent import layer_norm, recurrent_attention

    g = gen(B + T)
    rot = RotaryEmbedding.parse(rotary)
    dx, dy, e = torch.randn((h, d, N), generator=g), torch.randn((h, d, N), generator=g), torch.randn((h * N, d), generator=g)
    pdx, pdy, pe = (PackedWeights(w.to(DEV), dtype=kind) for w in (dx, dy, e))
    cur = layer_norm(torch.randn((B, 1, T, d), generator=g).to(DEV))
    rho = torch.randn((B, h, N, d), generator=g).to(DEV)
    x = packed_forward(cur, pdx)
    a = layer_norm(recurrent_attention(x, cur[:, 0], rho, build_freqs(N, 65536.0, rot, DEV), 7, rot,
                                       [0.5 ** (i + 1) for i in range(h)] if rotary == "alibi" else None))
    xy = packed_forward(a, pdy, gate=x)
    mixed = xy.permute(0, 2, 1, 3).reshape(B, T, h * N)
    out = product(mixed, pe)
    for b in range(B):
        for i in range(h):
            s, bound = definition(cur[b, 0].cpu(), dx[i], kind)
            close(x[b, i], np.maximum(s, 0), np.where(s < -bound, 0, bound), "x")
            s, bound = definition(a[b, i].cpu(), dy[i], kind)
            m = x[b, i].double().cpu().numpy()
            close(xy[b, i], m * np.maximum(s, 0), np.abs(m) * np.where(s < -bound, 0, bound) + 1.01 * 2.0**-24 * np.abs(m * s), "xy")
        close(out[b], *definition(mixed[b].cpu(), e, kind), "out")


def _big(kind=INT8, rotary=orc.ROPE, **kw):
    shape = orc.BDHShape(n_layer=2, n_embd=128, n_head=2, mlp_internal_dim_multiplier=8, vocab_size=40, rotary=rotary)
    model = build(shape, orc.init_weights(shape, 3), **kw)
    model.pack_projections(kind)
    return model


@pytest.mark.parametrize("kind", [INT8, BF16])
def test_prompts_of_many_tokens_leave_what_single_tokens_leave(kind):
    """The projections do not depend on how many rows go through them together: the same sums in 8 bits, and in bf16 sums of the
    same terms.  What differs are the orders of the state's sums, and where such a difference moves a value over a border, a step of
    8 (2^-7 of the row's largest value) or bf16: of 2 x 100 values of a row some do.  A test of the plumbing, hence the wide bound."""
    model = _big(kind)
    tokens = torch.randint(0, 40, (2, 9), generator=gen(2))
    one, many = model.init_state(), model.init_state()
    single = torch.cat([model.forward_with_state(tokens[:, t:t + 1], one) for t in range(9)], 1)
    together = model.forward_with_state(tokens, many)
    assert (single - together).abs().max() <= 0.02 * single.abs().max()
    assert one.position == many.position == 9


def test_by_products_shared_states_and_the_stateless_forward_run():
    model = _big()
    tokens = torch.randint(0, 40, (2, 5), generator=gen(4))
    state = model.init_state()
    plain = model.forward_with_state(tokens, state)
    seen = model.init_state()
    assert torch.equal(model.forward_with_state(tokens, seen, viz=True), plain)
    x_last, y_last, xy_last = (getattr(seen.layers[1].viz, n) for n in ("x_last", "y_last", "xy_last"))
    # y is made once more for the map, and the product of the two rounded once
    assert torch.allclose(x_last * y_last, xy_last, rtol=2.0**-23, atol=0)
    nxt = torch.randint(0, 40, (2, 1), generator=gen(5))
    shared = model.share_state(_copied(model, state), [1, 1], capacity=4)
    a, b = model.forward_shared(nxt, shared), model.forward_with_state(nxt, state)
    assert (a - b).abs().max() <= 0.02 * b.abs().max()
    fast = model.forward_fast(tokens)
    assert fast.shape == (2, 5, 40) and torch.isfinite(fast).all()


def _copied(model, state):
    other = model.init_state()
    model._ensure_state(other, state.storage.shape[1])
    other.storage.copy_(state.storage)
    other.position = state.position
    return other


def test_a_captured_step_keeps_the_weights_it_was_captured_with():
    model = _big()
    tokens = torch.randint(0, 40, (3, 6), generator=gen(6))
    state = model.init_state()
    _, nxt = model.forward_with_state(tokens, state, want_next=True)
    eager, t = _copied(model, state), nxt.clone()
    want = []
    for _ in range(6):
        logits, t = model.forward_with_state(t.reshape(3, 1), eager, want_next=True)
        want.append(logits)
    graph = model.capture_decode_step(state, nxt)
    model.pack_projections(None)  # the graph goes on with the packed weights
    for k in range(6):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graph.logits, want[k]), k
        other = model.init_state()
        model.forward_with_state(tokens, other)  # the program's own eager work in between
        torch.cuda.synchronize()


def test_what_is_refused():
    from burn_dragon_amd import BDH, BDHConfig, ffi
    from burn_dragon_amd.packed import PackedWeights

    model = _big()
    good = model.packed
    wrong = PackedWeights(torch.zeros(2, 128, 256, device=DEV))
    lib, check = model.ctx.lib, model.ctx.check
    for enc, encv, dec in ((None, good[1], good[2]), (good[0], None, None), (wrong, good[1], good[2]), (good[0], good[1], good[0])):
        with pytest.raises(ffi.BdhError):
            check(lib.bdh_model_set_packed(model.handle, *[None if w is None else w._ref for w in (enc, encv, dec)]))
    tokens = torch.randint(0, 40, (1, 4), generator=gen(7))
    before = model.forward_with_state(tokens, model.init_state())
    assert torch.equal(model.forward_with_state(tokens, model.init_state()), before)
    with pytest.raises(ValueError):
        model.pack_projections(torch.float16)
    from burn_dragon_amd.kernel.block_sparse import BlockPattern1d, BlockPattern2d, BlockSparseConfig

    model.kernel.enabled = True
    model.kernel.block_sparse = BlockSparseConfig(BlockPattern1d.from_blocks(64, [0]), BlockPattern2d.dense(64))
    with pytest.raises(ffi.BdhError):
        model.forward_fast(tokens)
