"""Many sequences of one prompt through a whole model: forward_shared and fork_shared next to forward_with_state on states
of their own, the sequences selected in between, and generate_samples, which runs all of it together.

Tolerance of the logits: 1e-3 of their largest magnitude, the bound of every f32 form of the model step here (a neuron
whose pre-activation is within rounding of the threshold may fire in one form and not in the other)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def bda():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device: the GPU tests must run on the MI355X box")
    import burn_dragon_amd

    return burn_dragon_amd


def _model(bda, rotary, dtype=0, d=128, mult=8, **more):
    cfg = bda.BDHConfig(n_layer=3, n_embd=d, n_head=4, mlp_internal_dim_multiplier=mult, vocab_size=69)
    cfg.fused_kernels.set_rotary_embedding(rotary)
    return bda.BDH(cfg, DEV, seed=3, rho_dtype=dtype, **more)


def _close(a, b, tol):
    assert (a - b).abs().max().item() <= tol * b.abs().max().item()


@pytest.mark.parametrize("rotary,lazy,dtype", [("rope", False, 0), ("alibi", False, 0), ("alibi", True, 0), ("pope", False, 0),
                                               ("rope", False, 1)])
def test_shared_sequences_equal_sequences_of_their_own(bda, rotary, lazy, dtype):
    model = _model(bda, rotary, dtype, alibi_lazy=lazy)
    tol = 1e-3 if dtype == 0 else 2e-2
    rng = np.random.default_rng(1)
    prompts = torch.from_numpy(rng.integers(0, 69, (2, 19)))
    counts, owner = [3, 1], [0, 0, 0, 1]
    state = model.init_state()
    model.forward_with_state(prompts, state)
    own = model.init_state()
    model.forward_with_state(prompts[owner], own)
    shared = model.share_state(state, counts, 14)
    assert shared.capacity == 16 and state.storage is None and state.position == 0
    for T in (5, 1, 1, 4, 1):
        tokens = torch.from_numpy(rng.integers(0, 69, (4, T)))
        logits, nxt = model.forward_shared(tokens, shared, want_next=True)
        want = model.forward_with_state(tokens, own)
        _close(logits, want, tol)
        assert torch.equal(nxt, logits[:, -1].argmax(-1))
    assert shared.position == own.position == 31 and shared.room == 4
    with pytest.raises(ValueError):
        model.forward_shared(torch.zeros((4, 5), dtype=torch.int64), shared)
    forked = model.fork_shared(shared)
    model.materialize_state(own)
    _close(forked.storage.float(), own.storage.float(), tol)
    tokens = torch.from_numpy(rng.integers(0, 69, (4, 3)))
    _close(model.forward_with_state(tokens, forked), model.forward_with_state(tokens, own), tol)


def test_selected_sequences_go_on_alike(bda):
    model = _model(bda, "rope")
    rng = np.random.default_rng(2)
    state = model.init_state()
    model.forward_with_state(torch.from_numpy(rng.integers(0, 69, (2, 8))), state)
    shared = model.share_state(state, [3, 2], 8)
    model.forward_shared(torch.from_numpy(rng.integers(0, 69, (5, 2))), shared)
    picked = model.select_shared(shared, [2, 0, 0, 4])
    assert picked.counts == [3, 1]
    with pytest.raises(ValueError):
        model.select_shared(shared, [3, 0])
    own = model.fork_shared(shared)
    few = model.select_sequences(own, [2, 0, 0, 4])
    tokens = torch.from_numpy(rng.integers(0, 69, (4, 1)))
    a, b = model.forward_shared(tokens, picked), model.forward_with_state(tokens, few)
    _close(a, b, 1e-3)
    before = own.storage.clone()
    assert model.select_sequences(own, [4, 3, -1, 1, 0]) is own
    assert torch.equal(own.storage[:, [0, 1, 3, 4]], before[:, [4, 3, 1, 0]]) and not own.storage[:, 2].any()


@pytest.mark.parametrize("rotary", ["rope", "alibi"])
def test_greedy_samples_equal_the_single_sequence(bda, rotary):
    """Greedy tokens of every sample against generate_tokens; runs past the shared capacity and through the fork.  The two
    may only part where the two largest logits are within rounding of each other, which the test looks up."""
    from burn_dragon_amd.generation import GenerationSettings, generate_samples, generate_tokens

    model = _model(bda, rotary, d=256, mult=4)
    prompt = [int(t) for t in np.random.default_rng(4).integers(0, 69, 21)]
    settings = GenerationSettings(max_new_tokens=30, top_k=1)
    want = generate_tokens(model, prompt, settings)[21:]
    got = generate_samples(model, prompt, 3, settings, capacity=12)
    for sample in got:
        assert len(sample) == 30
        if sample != want:
            i = next(i for i, (a, b) in enumerate(zip(sample, want)) if a != b)
            logits = model.forward(torch.tensor([prompt + want[:i]]))[0, -1]
            assert (logits[want[i]] - logits[sample[i]]).abs().item() <= 2e-3 * logits.abs().max().item()


def test_samples_with_rules_and_a_stop_token(bda):
    from burn_dragon_amd.generation import GenerationSettings, generate_samples
    from burn_dragon_amd.rules import pack_allowed

    model = _model(bda, "alibi", d=256, mult=4)
    prompt = list(range(10))
    allowed = torch.zeros(69, dtype=torch.bool)
    allowed[20:60] = True
    settings = GenerationSettings(max_new_tokens=50, temperature=1.0, top_k=None)

    def run(n, stop):
        rules = bda.LogitRules(repetition=1.3, presence=0.1, frequency=0.2, allowed=pack_allowed(allowed.to(DEV)))
        return generate_samples(model, prompt, n, settings, rules, stop, capacity=24,
                                generator=torch.Generator().manual_seed(5))

    free = run(6, None)
    assert all(len(s) == 50 and all(20 <= t < 60 for t in s) for s in free)
    assert len({tuple(s) for s in free}) > 1
    stop = free[0][9]  # a token that some samples draw
    ended = run(6, stop)
    for a, b in zip(ended, free):
        cut = b[:b.index(stop) + 1] if stop in b else b
        alike = min(16, len(a), len(cut))  # the batch changes after 16 tokens, and with it the order of sums
        assert stop not in a[:-1] and a[:alike] == cut[:alike]
    # never twice the same token under a frequency penalty that outweighs every logit
    rules = bda.LogitRules(frequency=1e6)
    for s in generate_samples(model, prompt, 4, GenerationSettings(max_new_tokens=40), rules, capacity=16):
        assert len(set(s)) == 40


def test_one_sample_one_token(bda):
    from burn_dragon_amd.generation import GenerationSettings, generate_samples

    model = _model(bda, "rope")
    for n in (1, 2):
        got = generate_samples(model, [3], n, GenerationSettings(max_new_tokens=1, top_k=1))
        assert [len(s) for s in got] == [1] * n
    assert generate_samples(model, [3], 2, GenerationSettings(max_new_tokens=0)) == [[], []]


def test_states_of_other_models_and_captures_are_refused(bda, monkeypatch):
    model, half, other = _model(bda, "rope"), _model(bda, "rope", 1), _model(bda, "rope", d=64)
    state = model.init_state()
    model.forward_with_state(torch.tensor([[1, 2, 3]]), state)
    shared = model.share_state(state, [2], 8)
    tokens = torch.tensor([[4], [5]])
    for m in (half, other):
        with pytest.raises(ValueError, match="another model"):
            m.forward_shared(tokens, shared)
        with pytest.raises(ValueError, match="another model"):
            m.fork_shared(shared)
    with monkeypatch.context() as p:
        p.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(ValueError, match="capture"):
            model.forward_shared(tokens, shared)
    assert shared.length == 0 and model.forward_shared(tokens, shared).shape == (2, 1, 69)


def test_states_with_logged_updates_are_flushed_before_they_are_shared_or_moved(bda):
    model, plain = _model(bda, "rope", d=256, mult=16, defer_updates=8), _model(bda, "rope", d=256, mult=16)
    rng = np.random.default_rng(6)
    prompts = torch.from_numpy(rng.integers(0, 69, (3, 7)))
    steps = torch.from_numpy(rng.integers(0, 69, (3, 3)))
    states = []
    for m in (model, plain):
        state = m.init_state()
        m.forward_with_state(prompts, state)
        for i in range(3):
            m.forward_with_state(steps[:, i:i + 1], state)
        states.append(state)
    assert states[0].logs is not None and states[0].logs.pending
    moved = [m.select_sequences(s, [2, 0]) for m, s in zip((model, plain), states)]
    shared = [m.share_state(s, [1, 2, 1], 4) for m, s in zip((model, plain), states)]
    tokens = torch.from_numpy(rng.integers(0, 69, (4, 1)))
    _close(*[m.forward_shared(tokens, s) for m, s in zip((model, plain), shared)], 1e-3)
    _close(*[m.forward_with_state(tokens[:2], s) for m, s in zip((model, plain), moved)], 1e-3)


def test_a_sample_of_which_the_rules_allow_nothing_ends(bda):
    """A row whose mask is empty from the start, one that a bias takes everything from, and rows that run out of allowed tokens
    as none may be said twice: each ends with what it was allowed, the others go on."""
    from burn_dragon_amd.generation import GenerationSettings, generate_samples
    from burn_dragon_amd.rules import pack_allowed

    model = _model(bda, "rope")
    allowed = torch.zeros((5, 69), dtype=torch.bool)
    for row, n in enumerate((0, 40, 5, 19, 69)):
        allowed[row, :n] = True
    bias = torch.zeros((5, 69))
    bias[4] = float("-inf")
    sizes = [0, 40, 5, 19, 0]
    for stop in (None, 68):
        rules = bda.LogitRules(frequency=float("inf"), bias=bias.to(DEV), allowed=pack_allowed(allowed.to(DEV)))
        got = generate_samples(model, [3, 1, 4], 5, GenerationSettings(max_new_tokens=60), rules, stop, capacity=12)
        assert [sorted(s) for s in got] == [list(range(n)) for n in sizes]
    one = bda.LogitRules(allowed=torch.zeros(3, dtype=torch.int32, device=DEV))
    assert generate_samples(model, [3], 2, GenerationSettings(max_new_tokens=3), one) == [[], []]


def test_positions_beyond_31_bits_are_refused(bda):
    """Positions are held in 32 bits beside a shared state: the last one that fits is rotated as sequences of their own rotate it, one
    more is refused and the state is not taken over.  Nothing is rotated by ALiBi."""
    model = _model(bda, "rope")
    state, own = model.init_state(), model.init_state()
    model.forward_with_state(torch.tensor([[1, 2, 3]]), state)
    model.forward_with_state(torch.tensor([[1, 2, 3], [1, 2, 3]]), own)
    state.position = own.position = 2**31 - 9
    for capacity in (9, 12, 100):
        with pytest.raises(ValueError, match="position"):
            model.share_state(state, [2], capacity)
    assert state.storage is not None and state.position == 2**31 - 9
    shared = model.share_state(state, [2], 8)
    for t in range(8):
        tokens = torch.tensor([[t], [9 - t]])
        _close(model.forward_shared(tokens, shared), model.forward_with_state(tokens, own), 1e-3)
    assert shared.position == own.position == 2**31 - 1 and shared.positions.tolist() == [2**31 - 1] * 2
    decaying = _model(bda, "alibi")
    state, own = decaying.init_state(), decaying.init_state()
    for s in (state, own):
        decaying.forward_with_state(torch.tensor([[1, 2, 3]]), s)
        s.position = 2**31 + 5
    shared = decaying.share_state(state, [1], 4)
    for t in range(3):
        _close(decaying.forward_shared(torch.tensor([[t]]), shared), decaying.forward_with_state(torch.tensor([[t]]), own), 1e-3)
    assert shared.position == 2**31 + 8


def _row_sets(n):
    """Tokens of a vocabulary of 300 that row i may say, disjoint, and the stop token"""
    sizes = [10, 25, 40, 55, 70, 12][:n]
    ends = np.cumsum(sizes)
    return [list(range(e - s, e)) for s, e in zip(sizes, ends)], 299


def _row_rules(bda, sets, stop):
    """Each row says its tokens once (a second time costs 1e6) and then, as its bias is lower than any logit, the stop token."""
    from burn_dragon_amd.rules import pack_allowed

    allowed = torch.zeros((len(sets), 300), dtype=torch.bool)
    for row, tokens in enumerate(sets):
        allowed[row, tokens] = allowed[row, stop] = True
    bias = torch.zeros(300)
    bias[stop] = -1e4
    return bda.LogitRules(frequency=1e6, bias=bias.to(DEV), allowed=pack_allowed(allowed.to(DEV)))


@pytest.mark.parametrize("rotary,lazy", [("rope", False), ("alibi", True)])
@pytest.mark.parametrize("capacity", [20, 4, 96])
@pytest.mark.parametrize("top_k", [1, None])
def test_rows_stay_their_own_as_others_leave(bda, rotary, lazy, capacity, top_k):
    """Six samples that may say disjoint sets of tokens, of six sizes: they leave the batch after 16, 32, 48, 64 and 80 draws, with
    shared states (capacity 96), with states of their own (4) and with both (20).  Every sample says exactly its set and the stop
    token; and walked again alone, with its own counts and its own variates, it draws the same tokens: greedy ones up to logits
    that are within the bound of each other (2e-3 of the largest), drawn ones between the tokens of its variate moved by twice that
    much either way (weights are then off by as much, relatively, and their sums too)."""
    from burn_dragon_amd.generation import (GenerationSettings, generate_samples, prefill_state, sample_from_logits,
                                            uniform_variates)

    cfg = bda.BDHConfig(n_layer=2, n_embd=128, n_head=4, mlp_internal_dim_multiplier=8, vocab_size=300)
    cfg.fused_kernels.set_rotary_embedding(rotary)
    model = bda.BDH(cfg, DEV, seed=3, alibi_lazy=lazy)
    sets, stop = _row_sets(6)
    prompt = [7, 250, 31, 8]
    settings = GenerationSettings(max_new_tokens=100, temperature=1.0, top_k=top_k)
    got = generate_samples(model, prompt, 6, settings, _row_rules(bda, sets, stop), stop, capacity,
                           torch.Generator().manual_seed(11))
    for sample, tokens in zip(got, sets):
        assert sample[-1] == stop and sorted(sample[:-1]) == tokens
    source = torch.Generator().manual_seed(11)
    variates = torch.cat([uniform_variates(96, DEV, source).reshape(16, 6) for _ in range(5)])
    for row, sample in enumerate(got):
        state, logits = prefill_state(model, prompt)
        left = set(sets[row])
        for step, token in enumerate(sample[:-1]):
            slack = 1e-3 * logits.abs().max().item()
            ruled = torch.full_like(logits, float("-inf"))
            index = torch.tensor(sorted(left), device=DEV)
            ruled[index] = logits[index]
            if top_k == 1:
                assert ruled[token] >= ruled.max() - 2 * slack
            else:
                u = variates[step, row]
                at = [sample_from_logits(model, ruled[None], 1.0, None, (u + m).clamp(0, 1 - 2**-24)[None]).item()
                      for m in (-4 * slack, 4 * slack)]
                assert at[0] <= token <= at[1], (row, step)
            left.remove(token)
            logits = model.forward_with_state(torch.tensor([[token]]), state)[0, -1]


@pytest.mark.parametrize("rotary,dtype,counts,T", [("rope", 0, [2, 1], 45), ("rope", 0, [2, 2], 20), ("alibi", 0, [4], 30),
                                                   ("pope", 0, [1, 2], 45), ("rope", 1, [2, 2], 20), ("rope", 1, [1, 2], 45)])
def test_a_follow_up_prompt_through_dense_products(bda, rotary, dtype, counts, T):
    """So many tokens that their products are dense ones, with the LayerNorm that a model takes of them: 4 heads of 1024 rows (PoPE
    2048) of 256 numbers, 2^20 multiplications a query; more than 32 queries a prompt and 2^25 multiplications, 2^27 where the
    prompts' counts differ.  Then single tokens, another such call, and the fork, next to states of their own."""
    model = _model(bda, rotary, dtype, d=256, mult=16)
    assert model.latent == 1024 and sum(counts) * T > 32 * len(counts) and sum(counts) * T > (32 if len(set(counts)) == 1 else 128)
    tol = 1e-3 if dtype == 0 else 2e-2
    rng = np.random.default_rng(12)
    B, owner = sum(counts), [g for g, n in enumerate(counts) for _ in range(n)]
    prompts = torch.from_numpy(rng.integers(0, 69, (len(counts), 11)))
    state, own = model.init_state(), model.init_state()
    model.forward_with_state(prompts, state)
    model.forward_with_state(prompts[owner], own)
    shared = model.share_state(state, counts, 2 * T + 3)
    for n in (T, 1, 1, T):
        tokens = torch.from_numpy(rng.integers(0, 69, (B, n)))
        logits, nxt = model.forward_shared(tokens, shared, want_next=True)
        _close(logits, model.forward_with_state(tokens, own), tol)
        assert torch.equal(nxt, logits[:, -1].argmax(-1))
    _close(model.fork_shared(shared).storage.float(), own.storage.float(), tol)
