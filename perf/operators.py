"""Many answers of one prompt, as operators that can be timed and compared.

Four kinds of call, each in a plain form of elementary torch operations and through burn_dragon_amd:

  read    attention of sequences that continue shared prompts: the state of a prompt is read once for all of its
          sequences, each adds its own tokens to it                        shared.shared_prefix_attention
  fork    the state of a prompt and a sequence's own tokens become a state of its own      shared.shared_prefix_fork
  slots   sequences of a batch forked, compacted and freed in the buffers that hold them   slots.copy_slots
  rules   penalties for repeated tokens, biases and masks on a step's logits               rules.count_tokens, apply_rules

Sizes: the default configuration (4 heads of 256 neurons, width 256), the many-neuron byte model (4 heads of 8192, width
256) and the largest model of the benchmark (8 heads of 16384, width 512); activations are relu(N(mu, 1)) of a stated
density (5 % as a trained model fires, half as a freshly initialised one does).
"""
from __future__ import annotations

import math
from statistics import NormalDist

import torch

own = False

DEVICE = "cuda:0"
THETA = 65536.0


def _read(name, counts, tokens, heads, latent, embd, rotary, state, capacity, shortest, longest, start, density):
    return {"name": name, "kind": "read", "counts": counts, "tokens": tokens, "heads": heads, "latent": latent,
            "embd": embd, "rotary": rotary, "state": state, "capacity": capacity, "shortest": shortest,
            "longest": longest, "start": start, "density": density}


def _fork(name, counts, heads, latent, embd, rotary, state, capacity, shortest, longest, density):
    return {"name": name, "kind": "fork", "counts": counts, "heads": heads, "latent": latent, "embd": embd,
            "rotary": rotary, "state": state, "capacity": capacity, "shortest": shortest, "longest": longest,
            "start": 500, "density": density}


def _slots(name, form, layers, slots, sources, heads, latent, embd, state, vocab):
    return {"name": name, "kind": "slots", "form": form, "layers": layers, "slots": slots, "sources": sources,
            "heads": heads, "latent": latent, "embd": embd, "state": state, "vocab": vocab}


def _rules(name, batch, vocab, prompt, bias, mask):
    return {"name": name, "kind": "rules", "batch": batch, "vocab": vocab, "prompt": prompt, "bias": bias, "mask": mask}


def listed():
    return [
        # four answers at the default configuration: the smallest step, all latency
        _read("read-default-b4", "4", 1, 4, 256, 256, "alibi", "f32", 32, 3, 21, 128, 0.5),
        # 32 answers of one prompt through the many-neuron byte model, in the middle of their answers
        _read("read-8192-b32", "32", 1, 4, 8192, 256, "rope", "f32", 64, 17, 60, 2048, 0.05),
        # answers of three prompts, some of them already finished, largest width, states in bf16
        _read("read-16384-bf16-b40", "20,7,13", 1, 8, 16384, 512, "rope", "bf16", 32, 0, 31, 100000, 0.05),
        # a follow-up question of 45 tokens to two conversations that six users share
        _read("read-8192-t45", "4,2", 45, 4, 8192, 256, "rope", "f32", 128, 0, 70, 777, 0.05),
        # answers that go on alone, default configuration
        _fork("fork-default-b4", "4", 4, 256, 256, "alibi", "f32", 32, 5, 32, 0.5),
        # 32 answers whose own tokens have filled the space for them
        _fork("fork-8192-b32", "32", 4, 8192, 256, "rope", "f32", 64, 64, 64, 0.05),
        # beams at the default configuration: losers are overwritten by winners in place, two hypotheses end
        _slots("slots-beams-16", "beams", 6, 16, 16, 4, 256, 256, "f32", 256),
        # one prompt's state for 16 answers that do not share it
        _slots("slots-fork-8192-b16", "fork", 2, 16, 1, 4, 8192, 256, "f32", 256),
        # 11 survivors of 24 conversations into a smaller batch, states in bf16
        _slots("slots-compact-bf16-24", "compact", 3, 11, 24, 8, 2048, 512, "bf16", 256),
        # one byte-level answer, a penalty for what it repeats: the smallest call
        _rules("rules-byte-b1", 1, 256, 0, False, False),
        # prompts are counted and the first token of each answer is constrained
        _rules("rules-prompt-b16", 16, 8192, 4001, True, True),
        # a large batch over a wide vocabulary of odd size
        _rules("rules-wide-b192", 192, 65601, 0, True, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["read", "read", "fork", "slots", "rules", "rules"])
    if kind == "rules":
        v = _log(rng, 60, 70000)
        return {k: x for k, x in _rules("", _log(rng, 1, max(1, min(256, 12000000 // v))), v,
                                        rng.choice([0, 0, _log(rng, 1, 5000)]), rng.random() < 0.5,
                                        rng.random() < 0.5).items() if k != "name"}
    heads = rng.choice([1, 2, 3, 4, 8])
    embd = 4 * _log(rng, 16, 128)
    if kind == "slots":
        form = rng.choice(["beams", "fork", "compact"])
        slots = _log(rng, 2, 40)
        latent = 2 * _log(rng, 30, 4100)
        layers = rng.randint(1, 4)
        while layers * slots * heads * latent * embd > 250e6:
            latent = latent // 4 * 2
        sources = slots if form == "beams" else rng.randint(1, 3) if form == "fork" else slots + rng.randint(0, 12)
        return {k: x for k, x in _slots("", form, layers, slots, sources, heads, latent, embd,
                                        rng.choice(["f32", "bf16"]), rng.choice([69, 256, 1000])).items() if k != "name"}
    counts = ",".join(str(_log(rng, 1, 24)) for _ in range(rng.choice([1, 1, 2, 3])))
    batch = sum(int(c) for c in counts.split(","))
    rotary = rng.choice(["rope", "rope", "alibi", "pope"])
    latent = 2 * _log(rng, 30, 8200)
    tokens = rng.choice([1, 1, 1, _log(rng, 2, 60)]) if kind == "read" else 0
    capacity = 4 * _log(rng, 4, 40)
    while batch * heads * latent * (capacity + (embd if kind == "fork" else 3 * tokens)) > 200e6:
        latent = latent // 4 * 2
    capacity = max(capacity, (tokens + 3) // 4 * 4 + 4)
    longest = rng.randint(0, capacity - tokens)
    shortest = rng.choice([longest, rng.randint(0, longest)])
    density = rng.choice([0.02, 0.05, 0.2, 0.5])
    state = rng.choice(["f32", "f32", "bf16"])
    if kind == "fork":
        return {k: x for k, x in _fork("", counts, heads, latent, embd, rotary, state, capacity, shortest, longest,
                                       density).items() if k != "name"}
    return {k: x for k, x in _read("", counts, tokens, heads, latent, embd, rotary, state, capacity, shortest, longest,
                                   _log(rng, 1, 200000), density).items() if k != "name"}


# ---- inputs -----------------------------------------------------------------------------

def _counts(case):
    return [int(c) for c in case["counts"].split(",")]


def _freqs(latent):
    """As the framework builds it for RoPE: neuron n turns by theta^-(even part of n / latent) / 2 pi of a circle per token."""
    n = torch.arange(latent, dtype=torch.float64)
    even = torch.floor(n / 2) * 2
    return (THETA ** (-even / latent) / (2 * math.pi)).to(torch.float32).to(DEVICE)


def _slopes(heads):
    return [2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)]


def _activations(gen, shape, density):
    mu = NormalDist().inv_cdf(density)
    return torch.relu(torch.randn(shape, device=DEVICE, generator=gen) + mu)


def _turn(x, freqs, positions, rotary):
    """Queries and keys of activations x [B,h,T,N] at positions [B,T]: the product of position and frequency is rounded to
    32 bits by definition (its whole turns are taken off, the angle of the rest is taken in 64 bits)."""
    if rotary == "alibi":
        return x
    raw = positions.to(torch.float32)[:, None, :, None] * freqs
    angle = (raw - torch.floor(raw)).to(torch.float64) * (2 * math.pi)
    c, s = torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)
    del raw, angle
    if rotary == "pope":
        m = torch.log(torch.exp(x) + 1.0)
        return torch.cat([m * c, m * s], dim=-1)
    other = torch.stack([-x[..., 1::2], x[..., 0::2]], dim=-1).reshape(x.shape)
    return x * c + other * s


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    kind = case["kind"]
    if kind == "rules":
        return _prepare_rules(case, gen)
    dtype = torch.float32 if case["state"] == "f32" else torch.bfloat16
    if kind == "slots":
        return _prepare_slots(case, gen, host, dtype)
    counts = _counts(case)
    B, h, N, d, S = sum(counts), case["heads"], case["latent"], case["embd"], case["capacity"]
    Nq = 2 * N if case["rotary"] == "pope" else N
    freqs = _freqs(N)
    lens = torch.randint(case["shortest"], case["longest"] + 1, (B,), generator=host)
    lens[torch.randint(0, B, (1,), generator=host)] = case["longest"]
    start = torch.randint(max(1, case["start"] // 2), case["start"] + 1, (len(counts),), generator=host)
    start = torch.repeat_interleave(start, torch.tensor(counts))
    rho = (0.3 * torch.randn((len(counts), h, Nq, d), device=DEVICE, generator=gen)).to(dtype)
    keys = torch.zeros((B, h, Nq, S), device=DEVICE)
    values = torch.zeros((B, S, d), device=DEVICE)
    values.normal_(generator=gen)
    at = torch.arange(S)
    for b in range(B):  # what each sequence has said so far; the rest of its space holds zeros
        n = int(lens[b])
        values[b, n:] = 0.0
        if n:
            x = _activations(gen, (1, h, n, N), case["density"])
            keys[b, :, :, :n] = _turn(x, freqs, (start[b] + at[:n])[None].to(DEVICE), case["rotary"])[0].transpose(1, 2)
    state = {"case": case, "counts": counts, "rho": rho, "keys": keys, "values": values,
             "lens": lens.to(DEVICE, torch.int32), "longest": case["longest"],
             "slopes": _slopes(h) if case["rotary"] == "alibi" else None}
    if kind == "read":
        T = case["tokens"]
        state["freqs"] = freqs
        state["positions"] = (start + lens).to(DEVICE, torch.int32)
        state["x"] = _activations(gen, (B, h, T, N), case["density"])
        state["v"] = torch.randn((B, T, d), device=DEVICE, generator=gen)
    return state


def _prepare_slots(case, gen, host, dtype):
    """Three buffers of a batch: the states [L, slots, h, N, d], the tokens seen [slots, V], the positions [slots]."""
    L, n, m, h, N, d, V = (case[k] for k in ("layers", "slots", "sources", "heads", "latent", "embd", "vocab"))
    src = [torch.randn((L, m, h, N, d), device=DEVICE, generator=gen, dtype=dtype),
           torch.randint(0, 50, (m, V), device=DEVICE, generator=gen, dtype=torch.int32),
           torch.randint(0, 5000, (m,), device=DEVICE, generator=gen, dtype=torch.int32)]
    if case["form"] == "beams":  # every winner stays where it is, the others become copies of winners, the last are freed
        stays = torch.rand(n, generator=host) < 0.5
        stays[int(torch.randint(0, n, (1,), generator=host))] = True
        winners = torch.nonzero(stays).reshape(-1)
        origin = winners[torch.randint(0, len(winners), (n,), generator=host)]
        origin = torch.where(stays, torch.arange(n), origin)
        losers = torch.nonzero(~stays).reshape(-1)[-2:]
        origin[losers] = -1
        dst = src
    else:
        if case["form"] == "fork":
            origin = torch.randint(0, m, (n,), generator=host)
        else:
            origin = torch.sort(torch.randperm(m, generator=host)[:n])[0]
        dst = [torch.empty((L, n, h, N, d), device=DEVICE, dtype=dtype), torch.empty((n, V), device=DEVICE, dtype=torch.int32),
               torch.empty((n,), device=DEVICE, dtype=torch.int32)]
    return {"case": case, "src": src, "dst": dst, "dims": [1, 0, 0], "origin": origin.to(DEVICE, torch.int32)}


def _prepare_rules(case, gen):
    B, V, P = case["batch"], case["vocab"], case["prompt"]

    def uniform(lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(shape, device=DEVICE, generator=gen)

    state = {"case": case, "logits": 3.0 * torch.randn((B, V), device=DEVICE, generator=gen),
             "repetition": uniform(1.0, 1.5, B), "presence": uniform(0.0, 0.8, B), "frequency": uniform(0.0, 0.3, B),
             "newest": torch.randint(0, V, (B,), device=DEVICE, generator=gen)}
    seen = torch.zeros((B, V), device=DEVICE, dtype=torch.int32)
    spoken = (V * torch.rand((B, 400), device=DEVICE, generator=gen) ** 3).to(torch.int64).clamp(0, V - 1)
    seen.scatter_add_(1, spoken, torch.ones_like(spoken, dtype=torch.int32))
    state["seen"] = seen
    if P:
        state["tokens"] = (V * torch.rand((B, P), device=DEVICE, generator=gen) ** 2).to(torch.int64).clamp(0, V - 1)
        state["lengths"] = torch.randint(1, P + 1, (B,), device=DEVICE, generator=gen, dtype=torch.int32)
    if case["bias"]:
        state["bias"] = torch.randn((B, V), device=DEVICE, generator=gen)
    if case["mask"]:  # bit v % 32 of word v / 32; the first sequence may say nothing at all
        words = torch.randint(-2**31, 2**31, (B, (V + 31) // 32), device=DEVICE, generator=gen, dtype=torch.int64)
        words[0] = 0
        state["allowed"] = words.to(torch.int32)
    return state


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"read": _own_read, "fork": _own_fork, "slots": _own_slots, "rules": _own_rules}[kind](state)
    return {"read": _plain_read, "fork": _plain_fork, "slots": _plain_slots, "rules": _plain_rules}[kind](state)


def _own_read(s):
    from burn_dragon_amd.shared import shared_prefix_attention

    out = shared_prefix_attention(s["x"], s["v"], s["rho"], s["keys"], s["values"], s["lens"], s["freqs"],
                                  positions=s["positions"], rotary_embedding=s["case"]["rotary"],
                                  alibi_slopes=s["slopes"], counts=s["counts"], longest=s["longest"])
    return [out, s["keys"], s["values"]]


def _own_fork(s):
    from burn_dragon_amd.shared import shared_prefix_fork

    return shared_prefix_fork(s["rho"], s["keys"], s["values"], s["lens"], rotary_embedding=s["case"]["rotary"],
                              alibi_slopes=s["slopes"], counts=s["counts"], longest=s["longest"])


def _own_slots(s):
    from burn_dragon_amd.slots import copy_slots

    copy_slots(list(zip(s["dst"], s["src"], s["dims"])), s["origin"])
    return s["dst"]


def _own_rules(s):
    from burn_dragon_amd.rules import LogitRules, apply_rules, count_tokens

    rules = LogitRules(s["repetition"], s["presence"], s["frequency"], s.get("bias"), s.get("allowed"))
    if "tokens" in s:
        count_tokens(s["tokens"], s["seen"], s["lengths"], prompt=True)
    return [apply_rules(s["logits"], rules, s["seen"], s["newest"]), s["seen"]]


def _decays(s, steps):
    """[h, *steps.shape]: the decay of each head over `steps` tokens, in 64 bits; ones where nothing decays."""
    if s["slopes"] is None:
        return None
    g = torch.exp(-torch.tensor(s["slopes"], dtype=torch.float32)).to(torch.float64).to(steps.device)
    return torch.exp(torch.log(g).reshape(-1, *[1] * steps.dim()) * steps.to(torch.float64)).to(torch.float32)


def _plain_read(s):
    case, x, v, keys, values = s["case"], s["x"], s["v"], s["keys"], s["values"]
    B, h, T, N = x.shape
    S, d = keys.shape[3], v.shape[2]
    steps = torch.arange(T, device=DEVICE)
    lens = s["lens"].to(torch.int64)
    q = _turn(x, s["freqs"], s["positions"].to(torch.int64)[:, None] + steps, case["rotary"])  # [B,h,T,Nq]
    place = lens[:, None] + steps  # [B,T]: where each new token goes, and how many came before it
    b_at = torch.arange(B, device=DEVICE)[:, None].expand(B, T)
    keys.permute(0, 3, 1, 2)[b_at, place] = q.permute(0, 2, 1, 3)
    values[b_at, place] = v
    out = torch.empty((B, h, T, d), device=DEVICE)
    first = 0
    for g, n in enumerate(s["counts"]):  # all rows of a prompt's sequences in one product
        rows = q[first:first + n].permute(1, 0, 2, 3).reshape(h, n * T, -1)
        out[first:first + n] = torch.matmul(rows, s["rho"][g].to(torch.float32)).reshape(h, n, T, d).permute(1, 0, 2, 3)
        first += n
    ago = place[:, :, None] - torch.arange(S, device=DEVICE)  # [B,T,S]
    scores = torch.matmul(q, keys) * (ago > 0)[:, None]
    if s["slopes"] is not None:
        out = out * _decays(s, place).permute(1, 0, 2)[..., None]
        scores = scores * _decays(s, ago.clamp(min=0)).permute(1, 0, 2, 3)
    return [out + torch.matmul(scores, values[:, None].expand(B, h, S, d).contiguous()), keys, values]


def _plain_fork(s):
    keys, values, lens = s["keys"], s["values"], s["lens"].to(torch.int64)
    B, h, Nq, S = keys.shape
    owner = torch.repeat_interleave(torch.arange(len(s["counts"])), torch.tensor(s["counts"])).to(DEVICE)
    ago = lens[:, None] - torch.arange(S, device=DEVICE)
    weighted = (values * (ago > 0)[..., None])[:, None].expand(B, h, S, values.shape[2])
    base = s["rho"].to(torch.float32)[owner]
    if s["slopes"] is not None:
        weighted = weighted * _decays(s, ago.clamp(min=0)).permute(1, 0, 2)[..., None]
        base = base * _decays(s, lens).permute(1, 0)[..., None, None]
    return (base + torch.matmul(keys, weighted.contiguous())).to(s["rho"].dtype)


def _plain_slots(s):
    origin = s["origin"].to(torch.int64)
    for dst, src, dim in zip(s["dst"], s["src"], s["dims"]):
        picked = src.index_select(dim, origin.clamp(min=0))
        shape = [1] * src.dim()
        shape[dim] = -1
        dst.copy_(torch.where((origin >= 0).reshape(shape), picked, torch.zeros((), dtype=src.dtype, device=DEVICE)))
    return s["dst"]


def _plain_rules(s):
    seen, z = s["seen"], s["logits"]
    B, V = z.shape
    if "tokens" in s:
        tokens = s["tokens"]
        inside = torch.arange(tokens.shape[1], device=DEVICE) < s["lengths"][:, None]
        hits = torch.zeros((B, V), device=DEVICE, dtype=torch.int32).scatter_add_(1, tokens, inside.to(torch.int32))
        seen.copy_(torch.where(hits > 0, seen | -2**31, seen))
    seen.scatter_add_(1, s["newest"][:, None], torch.ones((B, 1), device=DEVICE, dtype=torch.int32))
    times = (seen & 0x7FFFFFFF).to(torch.float32)
    r = s["repetition"][:, None]
    z = torch.where(seen != 0, torch.where(z > 0, z / r, z * r), z)
    z = z - (s["frequency"][:, None] * times + s["presence"][:, None] * (times > 0))
    if "bias" in s:
        z = z + s["bias"]
    if "allowed" in s:
        v = torch.arange(V, device=DEVICE)
        bit = (s["allowed"][:, v // 32] >> (v % 32)) & 1
        z = torch.where(bit != 0, z, torch.full((), -math.inf, device=DEVICE))
    return [z, seen]


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "rules":
        B, V, P = case["batch"], case["vocab"], case["prompt"]
        each = 4 + 4 + 4 + (4 if case["bias"] else 0) + (0.125 if case["mask"] else 0)
        return {"bytes": int(B * V * each + B * P * 4 + 20 * B), "flops": 6 * B * V}
    size = 4 if case["state"] == "f32" else 2
    if kind == "slots":
        slot = case["layers"] * case["heads"] * case["latent"] * case["embd"] * size + 4 * case["vocab"] + 4
        n = case["slots"]
        if case["form"] == "beams":  # half of the slots stay; of the others two are cleared, the rest are copies
            return {"bytes": int(slot * (n / 2 + max(1, n / 4))), "flops": 0}
        used = min(case["sources"], n)
        return {"bytes": int(slot * (used + n)), "flops": 0}
    counts = _counts(case)
    B, h, N, d = sum(counts), case["heads"], case["latent"], case["embd"]
    Nq = 2 * N if case["rotary"] == "pope" else N
    said = (case["shortest"] + case["longest"]) / 2
    p = case["density"]

    def used(tokens):  # share of the rows that some of so many tokens uses
        if case["rotary"] == "pope":
            return 1.0
        return 1 - (1 - p) ** (tokens * (2 if case["rotary"] == "rope" else 1))

    if kind == "fork":
        held = B * h * Nq * said * used(1)
        state = len(counts) * h * Nq * d + B * h * Nq * d
        return {"bytes": int(state * size + 4 * held + 4 * B * said * d), "flops": int(2 * held * d)}
    T = case["tokens"]
    rows = sum(used(n * T) for n in counts) * h * Nq
    mean = said + (T - 1) / 2
    bytes_ = rows * d * size + B * h * Nq * used(T) * said * 4 + 4 * B * (said + 2 * T) * d  # states, keys, values
    bytes_ += 4 * B * h * T * N + 4 * N + 4 * B * h * T * d + 4 * B * h * T * Nq * used(1)  # x, table, out, new keys
    flops = 2 * B * h * T * (Nq * used(1) * (d + mean) + mean * d)
    return {"bytes": int(bytes_), "flops": int(flops)}


# ---- the definitions in 64 bits ---------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"read": _exact_read, "fork": _exact_fork, "slots": _exact_slots, "rules": _exact_rules}[case["kind"]](state)


def _exact_read(s):
    """Token by token, as a sequence's own state would be walked: one product with the prompt's state, one with each key."""
    case = s["case"]
    B, h, T, N = s["x"].shape
    keys, values = s["keys"].to(torch.float64), s["values"].to(torch.float64)
    out = torch.zeros((B, h, T, s["v"].shape[2]), device=DEVICE, dtype=torch.float64)
    g_of = [g for g, n in enumerate(s["counts"]) for _ in range(n)]
    rate = torch.zeros(h, dtype=torch.float64, device=DEVICE)
    if s["slopes"] is not None:
        rate = torch.log(torch.exp(-torch.tensor(s["slopes"], dtype=torch.float32)).to(torch.float64)).to(DEVICE)
    lens, positions = s["lens"].tolist(), s["positions"].tolist()
    for g in range(len(s["counts"])):
        rho = s["rho"][g].to(torch.float64)
        for b in [b for b in range(B) if g_of[b] == g]:
            for t in range(T):
                k = lens[b] + t
                x = s["x"][b, :, t].to(torch.float64)
                if case["rotary"] != "alibi":
                    turns = s["freqs"] * torch.tensor(float(positions[b] + t), dtype=torch.float32, device=DEVICE)
                    angle = 2 * math.pi * torch.remainder(turns.to(torch.float64), 1.0)
                    if case["rotary"] == "pope":
                        m = torch.log1p(torch.exp(x))
                        x = torch.cat((m * angle.cos(), m * angle.sin()), 1)
                    else:
                        y = torch.empty_like(x)
                        y[:, 0::2] = x[:, 0::2] * angle[0::2].cos() - x[:, 1::2] * angle[0::2].sin()
                        y[:, 1::2] = x[:, 1::2] * angle[1::2].cos() + x[:, 0::2] * angle[1::2].sin()
                        x = y
                row = torch.bmm(x[:, None], rho)[:, 0] * torch.exp(rate * k)[:, None]
                if k:
                    back = torch.arange(k, 0, -1, device=DEVICE, dtype=torch.float64)
                    w = torch.bmm(x[:, None], keys[b, :, :, :k].contiguous())[:, 0] * torch.exp(rate[:, None] * back)
                    row = row + w @ values[b, :k]
                out[b, :, t] = row
                keys[b, :, :, k] = x
                values[b, k] = s["v"][b, t].to(torch.float64)
    return [out, keys, values]


def _exact_fork(s):
    """The states walked token by token."""
    rate = None
    if s["slopes"] is not None:
        rate = torch.exp(-torch.tensor(s["slopes"], dtype=torch.float32)).to(torch.float64).to(DEVICE)[:, None, None]
    rows, first = [], 0
    for g, n in enumerate(s["counts"]):
        for b in range(first, first + n):
            rho = s["rho"][g].to(torch.float64)
            for t in range(int(s["lens"][b])):
                rho = torch.addcmul(rho, s["keys"][b, :, :, t, None].to(torch.float64), s["values"][b, t].to(torch.float64))
                if rate is not None:
                    rho = rho * rate
            rows.append(rho)
        first += n
    return torch.stack(rows)


def _exact_slots(s):
    out = []
    for dst, src, dim in zip(s["dst"], s["src"], s["dims"]):
        pieces = [src.select(dim, o).clone() if o >= 0 else torch.zeros_like(src.select(dim, 0)) for o in s["origin"].tolist()]
        whole = torch.stack(pieces, dim)
        out.append(whole.to(torch.float64) if whole.is_floating_point() else whole)
    return out


def _exact_rules(s):
    B, V = s["logits"].shape
    z, seen = s["logits"].to(torch.float64), s["seen"].clone()
    for b in range(B):
        if "tokens" in s:
            said = torch.unique(s["tokens"][b, :int(s["lengths"][b])])
            seen[b, said] = seen[b, said] | -2**31
        seen[b, int(s["newest"][b])] += 1
        n = torch.remainder(seen[b].to(torch.int64), 2**31).to(torch.float64)
        r = s["repetition"][b].to(torch.float64)
        met = torch.nonzero(seen[b]).reshape(-1)
        z[b, met] = torch.maximum(z[b, met], torch.zeros_like(r)) / r + torch.minimum(z[b, met], torch.zeros_like(r)) * r
        z[b] -= s["frequency"][b].to(torch.float64) * n + s["presence"][b].to(torch.float64) * n.clamp(max=1)
        if "bias" in s:
            z[b] += s["bias"][b].to(torch.float64)
        if "allowed" in s:
            words = s["allowed"][b].to(torch.int64)
            bits = torch.stack([(words >> i) & 1 for i in range(32)], 1).reshape(-1)[:V]
            z[b][bits == 0] = -math.inf
    return [z, seen]
