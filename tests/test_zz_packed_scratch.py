"""Captured steps of models whose later calls need more scratch than the ones before the capture, and packed weights that are replaced while
a stream reads them."""
import pytest
import torch

from oracle import bdh_oracle as orc

from .test_gpu_packed import BF16, DEV, INT8, gen
from .test_zz_packed_model import _copied, build
from .test_zz_packed_prompts import _model

pytestmark = pytest.mark.gpu


def _steps(model, state, token, n):
    """The logits of n greedy steps, eagerly, on a copy of the state."""
    own, t, out = _copied(model, state), token.clone(), []
    for _ in range(n):
        logits, t = model.forward_with_state(t.reshape(-1, 1), own, want_next=True)
        out.append(logits)
    return out


def _goes_on(model, state, token, later):
    """A step captured, `later` run, and the step replayed with more calls in between: the logits are the eager ones."""
    want = _steps(model, state, token, 6)
    graph = model.capture_decode_step(state, token)
    for k in range(6):
        later(k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graph.logits, want[k]), k


@pytest.mark.parametrize("kind", [INT8, BF16])
def test_a_captured_step_of_f32_weights_goes_on_beside_packed_prompts(kind):
    shape = orc.BDHShape(n_layer=2, n_embd=256, n_head=4, mlp_internal_dim_multiplier=128, vocab_size=40, rotary=orc.ROPE)
    model = build(shape, orc.init_weights(shape, 4))
    tokens = torch.randint(0, 40, (1, 64), generator=gen(8))
    state = model.init_state()
    _, token = model.forward_with_state(tokens, state, want_next=True)

    def later(k):
        if k == 0:
            model.pack_projections(kind)
        model.forward_with_state(tokens if k < 3 else tokens.repeat(1, k), model.init_state())

    _goes_on(model, state, token, later)


def test_a_captured_step_of_a_small_packed_model_goes_on_beside_longer_prompts():
    shape = orc.BDHShape(n_layer=2, n_embd=256, n_head=4, mlp_internal_dim_multiplier=4, vocab_size=40, rotary=orc.ROPE)
    model = build(shape, orc.init_weights(shape, 5))
    model.pack_projections()
    tokens = torch.randint(0, 40, (3, 20), generator=gen(9))
    state = model.init_state()
    _, token = model.forward_with_state(tokens, state, want_next=True)
    _goes_on(model, state, token, lambda k: model.forward_with_state(tokens.repeat(1, 1 + 10 * k), model.init_state()))


def test_weights_that_are_replaced_while_a_stream_reads_them():
    """Memory of the old packed weights is not given to the stream that made them while another one's calls are queued."""
    model = _model(INT8, 4, 256, 1024)
    tokens = torch.randint(0, 50, (2, 100), device=DEV)
    want = model.forward_with_state(tokens, model.init_state())
    torch.cuda.synchronize()
    old = [(w.data.data_ptr(), w.data.numel()) for w in model.packed]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        model.forward_with_state(tokens, model.init_state())
        torch.cuda.synchronize()
        torch.cuda._sleep(1_000_000_000)
        held = torch.cuda.Event()
        held.record()
        got = model.forward_with_state(tokens, model.init_state())
        model.pack_projections(None)
    taken = [torch.full((n,), 99, device=DEV, dtype=torch.uint8) for _, n in old for _ in range(2)]
    places = {t.data_ptr() for t in taken}
    assert not held.query(), "the wait was too short to show anything"
    torch.cuda.synchronize()
    assert not places & {p for p, _ in old}
    assert torch.equal(got, want)
