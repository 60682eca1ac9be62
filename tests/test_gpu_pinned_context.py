"""Contexts that keep a stream of their own: what the wrappers fill or copy on their way to a call is made on that stream, and what they
allocate is not handed out again before the call has read it.  One of the two streams waits (torch.cuda._sleep, a bounded
spin) while the other goes on."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WAIT = 1_000_000_000  # cycles, 0.4 s: a call takes less than a millisecond


@pytest.fixture(scope="module")
def bda():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device: the GPU tests must run on the MI355X box")
    import burn_dragon_amd

    return burn_dragon_amd


@pytest.fixture()
def pinned(bda):
    side = torch.cuda.Stream()
    ctx = bda.ffi.Context(0, side.cuda_stream)
    yield ctx, side
    torch.cuda.synchronize()
    ctx.close()


def _late(side, call):
    """What `call` leaves on the pinned stream while torch's own stream has not got anywhere."""
    for tensor in (torch.full((64,), float("nan"), device=DEV), torch.full((64,), -7, device=DEV)):
        del tensor  # what an allocation on this stream would find
    torch.cuda.synchronize()
    torch.cuda._sleep(WAIT)
    held = torch.cuda.Event()
    held.record()
    result = call()
    side.synchronize()
    copy = [t.clone() for t in result] if not held.query() else None
    assert copy is not None, "the wait was too short to show anything"
    torch.cuda.synchronize()
    return copy


def test_penalties_and_newest_tokens_of_a_pinned_context(bda, pinned):
    from burn_dragon_amd.rules import LogitRules, apply_rules

    ctx, side = pinned
    gen = torch.Generator(DEV).manual_seed(1)
    z = torch.randn((6, 300), device=DEV, generator=gen)
    seen = torch.randint(0, 3, (6, 300), device=DEV, generator=gen, dtype=torch.int32)
    newest = torch.randint(0, 300, (6, 4), device=DEV, generator=gen)
    rules = LogitRules(repetition=1.5, presence=0.25, frequency=0.5)
    ours, theirs = seen.clone(), seen.clone()
    want = apply_rules(z, rules, ours, newest[:, 1])
    rows = newest[:, 2].contiguous().reshape(2, 3).t()  # of rows that lie apart, and of another shape
    also = apply_rules(z, rules, ours, rows)
    torch.cuda.synchronize()

    def call():
        a = apply_rules(z, rules, theirs, newest[:, 1], ctx=ctx)
        return a, apply_rules(z, rules, theirs, rows, ctx=ctx)

    got = _late(side, call)
    assert torch.equal(got[0], want) and torch.equal(got[1], also) and torch.equal(theirs, ours)


def test_frequencies_of_another_shape(bda, pinned):
    from burn_dragon_amd.shared import shared_prefix_attention

    ctx, side = pinned
    gen = torch.Generator(DEV).manual_seed(2)
    B, h, N, d, S = 3, 2, 64, 32, 8
    x, v = torch.randn((B, h, 1, N), device=DEV, generator=gen).relu(), torch.randn((B, 1, d), device=DEV, generator=gen)
    rho = torch.randn((1, h, N, d), device=DEV, generator=gen)
    freqs = torch.rand((2, N // 2), device=DEV, generator=gen).t()  # rows that lie apart: [N/2, 2]
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    keys = [torch.zeros((B, h, N, S), device=DEV) for _ in range(2)]
    values = [torch.zeros((B, S, d), device=DEV) for _ in range(2)]
    want = shared_prefix_attention(x, v, rho, keys[0], values[0], lens, freqs, position=9)
    got, = _late(side, lambda: [shared_prefix_attention(x, v, rho, keys[1], values[1], lens, freqs, position=9, ctx=ctx)])
    assert torch.equal(got, want) and torch.equal(keys[0], keys[1])


def test_a_listed_origin_lives_until_the_slots_are_moved(bda, pinned):
    from burn_dragon_amd.slots import KEEP, copy_slots

    ctx, side = pinned
    a = torch.arange(5 * 40, device=DEV, dtype=torch.float32).reshape(5, 40)
    before = a.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(WAIT)
        held = torch.cuda.Event()
        held.record()
    copy_slots([(a, a, 0)], [4, 3, -1, 0, 2], ctx=ctx)
    others = [torch.full((5,), KEEP, device=DEV, dtype=torch.int32) for _ in range(64)]
    torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    assert torch.equal(a[[0, 1, 3, 4]], before[[4, 3, 0, 2]]) and not a[2].any() and len(others) == 64


def test_samples_of_a_model_whose_context_keeps_a_stream(bda):
    """The loop's own torch work runs on the stream of the model's context."""
    from burn_dragon_amd.generation import GenerationSettings, generate_samples

    cfg = bda.BDHConfig(n_layer=2, n_embd=64, n_head=2, mlp_internal_dim_multiplier=4, vocab_size=69)
    settings = GenerationSettings(max_new_tokens=40, temperature=1.0)
    rules = bda.LogitRules(repetition=1.2, frequency=0.3)
    model = bda.BDH(cfg, DEV, seed=3)

    def run():
        return generate_samples(model, [5, 6, 7], 4, settings, rules, 11, 12, torch.Generator().manual_seed(3))

    want = run()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    shared_ctx, follow = model.ctx, model.ctx._follow
    try:
        shared_ctx.set_stream(side.cuda_stream, pin=True)
        torch.cuda._sleep(WAIT)
        held = torch.cuda.Event()
        held.record()
        got = run()
        assert not held.query(), "the wait was too short to show anything"
    finally:
        torch.cuda.synchronize()
        shared_ctx._follow = follow
        shared_ctx.lib
    assert got == want
