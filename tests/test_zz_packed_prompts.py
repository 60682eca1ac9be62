"""Prompts through models whose projections are packed, long enough for tiles and parts of k, against the model's operators called one
after the other: embedding and LayerNorm, D_x, the state step, D_y with its gate, E.  The sums of the state step and the LayerNorms
may come in another order there.  Where such a difference moves a value over a border between two whole numbers (or two bf16
numbers), a product changes by a step of 2^-7 of its row's largest term; a few of a row's hundreds of values do.  Hence 2 % of the
largest logit, per token; a wrong row, gate or head is off by as much as the logits are."""
import pytest
import torch

from oracle import bdh_oracle as orc

from .packed_shapes import PROMPTS
from .test_gpu_packed import BF16, DEV, INT8, gen
from .test_zz_packed_model import build

pytestmark = pytest.mark.gpu


def _model(kind, h, d, N, layers=2, **kw):
    shape = orc.BDHShape(n_layer=layers, n_embd=d, n_head=h, mlp_internal_dim_multiplier=h * N // d, vocab_size=50, rotary=kw.pop("rotary", orc.ROPE))
    assert shape.latent_per_head == N
    model = build(shape, orc.init_weights(shape, N + d), **kw)
    if kind is not None:
        model.pack_projections(kind)
    return model


def _operators(model, tokens, attention):
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward
    from burn_dragon_amd.packed import product
    from burn_dragon_amd.recurrent import layer_norm

    (B, T), h, d, N = tokens.shape, model.n_head, model.n_embd, model.latent
    dx, dy, e = model.packed
    cur = layer_norm(model.params["embed"][tokens.to(DEV)].reshape(B, 1, T, d).contiguous())
    xs = []
    for _ in range(model.n_layer):
        x = packed_forward(cur, dx)
        xs.append(x)
        xy = packed_forward(layer_norm(attention(x, cur)), dy, gate=x)
        out = product(xy.permute(0, 2, 1, 3).reshape(B, T, h * N), e)
        cur = layer_norm(cur + layer_norm(out.reshape(B, 1, T, d)))
    return (cur.reshape(B * T, d).double() @ model.params["lm_head"].double()).reshape(B, T, -1), xs


def _same(got, want):
    off = (got.double() - want).abs().amax(-1) / want.abs().amax(-1)
    assert off.max() <= 0.02, (off.max().item(), int((off > 0.02).sum()))


@pytest.mark.parametrize("kind,h,d,N,B,T", PROMPTS)
def test_a_prompt_is_its_operators(kind, h, d, N, B, T):
    from burn_dragon_amd import RotaryEmbedding
    from burn_dragon_amd.kernel.block_sparse import BlockPattern2d
    from burn_dragon_amd.kernel.linear_attention import build_freqs, fused_state_aligned
    from burn_dragon_amd.recurrent import recurrent_attention

    model = _model({1: BF16, 2: INT8}[kind], h, d, N)
    tokens = torch.randint(0, 50, (B, T), generator=gen(T))
    freqs = build_freqs(N, 65536.0, RotaryEmbedding.ROPE, DEV)
    rho = []

    def step(x, cur):
        rho.append(torch.zeros((B, h, N, d), device=DEV))
        return recurrent_attention(x, cur[:, 0], rho[-1], freqs, 0, RotaryEmbedding.ROPE)

    want, xs = _operators(model, tokens, step)
    state = model.init_state()
    tap = torch.empty((model.n_layer, B, h, T, N), device=DEV)
    _same(model.forward_with_state(tokens, state, x_tap=tap), want)
    assert torch.equal(tap[0], xs[0])  # the first D_x has the same rows
    for l in range(model.n_layer):
        assert (state.storage[l] - rho[l]).abs().max() <= 0.02 * rho[l].abs().max()
    _same(model.forward_with_state(tokens, model.init_state()), want)  # without by-products
    fast, _ = _operators(model, tokens, lambda x, cur: fused_state_aligned(x, cur, freqs, None, BlockPattern2d.dense(1), RotaryEmbedding.ROPE))
    _same(model.forward_fast(tokens), fast)


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("d,N,T", [(256, 1024, 350), (260, 910, 600)])
def test_maps_of_a_long_prompt(d, N, T, kind):
    """The by-products are those of the last token of the first sequence."""
    model = _model(kind, 2, d, N)
    tokens = torch.randint(0, 50, (2, T), generator=gen(3))
    state, tap = model.init_state(), torch.empty((2, 2, 2, T, N), device=DEV)
    model.forward_with_state(tokens, state, x_tap=tap, viz=True)
    for l, layer in enumerate(state.layers):
        maps = layer.viz
        assert torch.equal(maps.x_last.reshape(2, N), tap[l, 0, :, -1])
        # y is made once more for the map, and the product of the two is rounded once (half a step each in bf16's f32 sums' order)
        least = 2.0**-22 * maps.xy_last.abs().max()
        assert ((maps.x_last * maps.y_last - maps.xy_last).abs() <= (2.0**-23 if kind is INT8 else 2.0**-14) * maps.xy_last.abs() + least).all()
        assert maps.xy_last.abs().max() > 0


def _logits(model, tokens, steps):
    state = model.init_state()
    out = [model.forward_with_state(tokens, state)]
    out += [model.forward_with_state(t, state) for t in steps]
    model.materialize_state(state)
    return out, state


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("rotary,options", [(orc.ROPE, {"defer_updates": 4}), (orc.ALIBI, {"alibi_lazy": True})])
def test_packed_models_with_deferred_updates_and_decay(rotary, options, kind):
    """A prompt and ten single tokens, against the packed model that updates and decays its state at once."""
    tokens = torch.randint(0, 50, (2, 90), generator=gen(4))
    steps = [torch.randint(0, 50, (2, 1), generator=gen(5 + i)) for i in range(10)]
    want, state = _logits(_model(kind, 4, 256, 256, rotary=rotary), tokens, steps)
    got, mine = _logits(_model(kind, 4, 256, 256, rotary=rotary, **options), tokens, steps)
    for a, b in zip(got, want):
        _same(a, b.double())
    assert (mine.storage - state.storage).abs().max() <= 0.02 * state.storage.abs().max() and mine.position == state.position
