"""Projections through weights that are packed for the matrix cores, as operators that can be timed and compared.

Three kinds of call, each in a plain form of elementary torch operations and through burn_dragon_amd:

  product   rows times weights: output heads, the encoder E                                 packed.product
  lowrank   the ReLU low-rank projections D_x and D_y: heads, threshold, gate               kernel.relu_lowrank.packed_forward
  grouped   rows sorted by the weights they meet, groups of ragged sizes                    packed.grouped_product

Weights are held in 8-bit integers with a scale for each output channel, or in bf16.  With 8-bit weights each row of the
input is brought to 8-bit integers with a scale of its own: of a largest magnitude a, the scale is a / 127 and a value x
becomes the whole number nearest to x * (127 / a), each of these operations rounded to 32 bits by definition; weights go by
the same rule along the inner dimension.  With bf16 weights the input is rounded to bf16.

Sizes: the default configuration (4 heads of 256 neurons, width 256), the many-neuron byte model (4 heads of 8192, width
256), the largest model of the benchmark (8 heads of 16384, width 512), and generic ones for the groups.
"""
from __future__ import annotations

import math
from statistics import NormalDist

import torch

own = False

DEVICE = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"f32": F32, "bf16": BF16}


def _product(name, rows, inner, outer, weights, x, out, density):
    return {"name": name, "kind": "product", "rows": rows, "inner": inner, "outer": outer, "weights": weights, "x": x,
            "out": out, "density": density}


def _lowrank(name, batch, tokens, heads, embd, latent, shared, gated, weights, x, out):
    return {"name": name, "kind": "lowrank", "batch": batch, "tokens": tokens, "heads": heads, "embd": embd, "latent": latent,
            "shared": shared, "gated": gated, "weights": weights, "x": x, "out": out}


def _grouped(name, rows, groups, inner, outer, skew, spare, weights, x, out):
    return {"name": name, "kind": "grouped", "rows": rows, "groups": groups, "inner": inner, "outer": outer, "skew": skew,
            "spare": spare, "weights": weights, "x": x, "out": out}


def listed():
    return [
        # the output head of the default configuration, one token: all latency
        _product("head-default-b1", 1, 256, 256, "int8", "f32", "f32", 1.0),
        # the encoder E of the many-neuron byte model in a decode step of 32 sequences: a long inner dimension, few rows
        _product("encoder-8192-b32", 32, 32768, 256, "int8", "f32", "f32", 0.05),
        # the same of the largest model for 2048 tokens of a prompt: reading the activations counts
        _product("encoder-16384-t2048", 2048, 131072, 512, "int8", "bf16", "f32", 0.05),
        # a wide vocabulary of odd size for 192 sequences
        _product("head-wide-b192", 192, 512, 65601, "bf16", "f32", "f32", 1.0),
        # D_x of the default configuration, four sequences decoding
        _lowrank("dx-default-b4", 4, 1, 4, 256, 256, True, False, "int8", "f32", "f32"),
        # D_y of the many-neuron byte model, eight sequences decoding: the weights are streamed once
        _lowrank("dy-8192-b8", 8, 1, 4, 256, 8192, False, True, "int8", "f32", "f32"),
        # D_x of the largest model for a prompt of 1500 tokens whose state step takes bf16: writing the activations counts
        _lowrank("dx-16384-t1500", 1, 1500, 8, 512, 16384, True, False, "int8", "f32", "bf16"),
        # D_y of two prompts of 777 tokens, bf16 weights
        _lowrank("dy-8192-t777", 2, 777, 4, 256, 8192, False, True, "bf16", "f32", "f32"),
        # D_x of three checkpoints of the default configuration that share a batch of 16 sequences
        _grouped("grouped-default-b16", 16, 3, 256, 1024, 1.0, 2, "int8", "f32", "f32"),
        # 64 rows dealt to 64 groups of weights, some of which get none: weights are streamed
        _grouped("grouped-64-b64", 64, 64, 2048, 1536, 0.7, 0, "bf16", "bf16", "bf16"),
        # a prompt's rows dealt to 24 groups of very different sizes
        _grouped("grouped-24-t8191", 8191, 24, 1024, 2816, 1.2, 37, "int8", "bf16", "bf16"),
        # a long prompt over eight groups, bf16 throughout: bound by the matrix cores
        _grouped("grouped-8-t16384", 16384, 8, 2048, 2048, 0.3, 0, "bf16", "bf16", "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _nameless(case):
    return {k: v for k, v in case.items() if k != "name"}


def draw(rng):
    kind = rng.choice(["product", "lowrank", "grouped"])
    weights = rng.choice(["int8", "int8", "bf16"])
    x, out = rng.choice(["f32", "f32", "bf16"]), rng.choice(["f32", "bf16"])
    if kind == "product":
        rows, inner, outer = _log(rng, 1, 8192), _log(rng, 16, 131072), _log(rng, 16, 66000)
        while inner * outer > 7e7 or rows * inner > 2.6e8 or rows * outer > 1.5e8 or 2 * rows * inner * outer > 2.6e11:
            rows, inner, outer = (rows * 3 + 3) // 4, (inner * 3 + 3) // 4, (outer * 3 + 3) // 4
        return _nameless(_product("", rows, inner, outer, weights, x, out, rng.choice([0.05, 0.5, 1.0])))
    if kind == "lowrank":
        heads, embd, latent = rng.choice([1, 2, 3, 4, 8]), 4 * _log(rng, 16, 128), _log(rng, 60, 16384)
        batch = _log(rng, 1, 64)
        tokens = rng.choice([1, _log(rng, 2, 2000)])
        while heads * embd * latent > 7e7 or batch * tokens * heads * latent > 1.5e8:
            batch, tokens, latent = (batch * 3 + 3) // 4, (tokens * 3 + 3) // 4, (latent * 9 + 9) // 10
        shared = rng.random() < 0.5
        return _nameless(_lowrank("", batch, tokens, heads, embd, latent, shared, rng.random() < (0.2 if shared else 0.8), weights,
                                  x, out))
    rows, groups, inner, outer = _log(rng, 1, 16384), _log(rng, 1, 128), _log(rng, 32, 4096), _log(rng, 32, 8192)
    while groups * inner * outer > 2.1e8 or rows * outer > 1.0e8 or 2 * rows * inner * outer > 1.5e11:
        rows, inner, outer = (rows * 7 + 7) // 8, (inner * 7 + 7) // 8, (outer * 7 + 7) // 8
    return _nameless(_grouped("", rows, groups, inner, outer, rng.choice([0.0, 0.5, 1.2]), rng.choice([0, 0, 5]), weights, x, out))


# ---- inputs -----------------------------------------------------------------------------

def _scaled(amax):
    """Scales for the largest magnitudes `amax`, and what values are multiplied by; nothing is held where the scale would be
    subnormal.  Quotients in 64 bits, rounded once: torch divides 32-bit numbers by way of a rounded reciprocal."""
    fits = amax >= 2.0 ** -118
    safe = torch.where(fits, amax, torch.ones((), device=amax.device)).to(torch.float64)
    nothing = torch.zeros((), device=amax.device)
    return torch.where(fits, (safe / 127.0).to(F32), nothing), torch.where(fits, (127.0 / safe).to(F32), nothing)


def _to_int8(x, dim):
    """x in 32 bits -> the whole numbers as f32, and the scales (with `dim` kept)."""
    amax = x.abs().amax(dim, keepdim=True)
    scale, up = _scaled(amax)
    return torch.round(x * up), scale


def _weights(gen, groups, inner, outer):
    """[G,K,N] as a trained projection: channels of different magnitudes."""
    w = 0.02 * torch.randn((groups, inner, outer), device=DEVICE, generator=gen)
    return w * (0.5 + torch.rand((groups, 1, outer), device=DEVICE, generator=gen))


def _rows(gen, shape, kind, density):
    """Activations: relu(N(mu, 1)) of a stated density, or rows that come out of a LayerNorm."""
    if density < 1.0:
        return torch.relu(torch.randn(shape, device=DEVICE, generator=gen) + NormalDist().inv_cdf(density)).to(TYPES[kind])
    return torch.randn(shape, device=DEVICE, generator=gen).to(TYPES[kind])


def _sizes(rows, groups, skew, host):
    """How many rows each group gets: shares that fall as a power of the group's rank, in random order."""
    share = torch.arange(1, groups + 1, dtype=torch.float64) ** -skew
    share = share[torch.randperm(groups, generator=host)]
    picked = torch.multinomial(share, rows, replacement=True, generator=host)
    return torch.bincount(picked, minlength=groups)


def _dense(case):
    """The weights' [groups, inner, outer]."""
    if case["kind"] == "lowrank":
        return case["heads"], case["embd"], case["latent"]
    return case.get("groups", 1), case["inner"], case["outer"]


def _prepared(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    w = _weights(gen, *_dense(case))
    state = {"case": case}
    if case["kind"] == "product":
        state["x"] = _rows(gen, (case["rows"], case["inner"]), case["x"], case["density"])
    elif case["kind"] == "lowrank":
        B, T, h, N = case["batch"], case["tokens"], case["heads"], case["latent"]
        state["x"] = _rows(gen, (B, 1 if case["shared"] else h, T, case["embd"]), case["x"], 1.0)
        if case["gated"]:
            state["gate"] = _rows(gen, (B, h, T, N), case["x"], 0.05)
    else:
        M, N = case["rows"], case["outer"]
        sizes = _sizes(M - min(case["spare"], M - 1), case["groups"], case["skew"], host)
        state["x"] = _rows(gen, (M, case["inner"]), case["x"], 1.0)
        state["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).to(DEVICE, torch.int32)
        state["longest"] = int(sizes.max())
        state["out"] = torch.zeros((M, N), device=DEVICE, dtype=TYPES[case["out"]])  # rows of no group stay as they are
    return state, w


def prepare(case, seed):
    """The weights are laid out once, as a program does that loads a checkpoint."""
    state, w = _prepared(case, seed)
    if own:
        from burn_dragon_amd.packed import PackedWeights

        state["weights"] = PackedWeights(w, dtype=torch.int8 if case["weights"] == "int8" else BF16)
    elif case["weights"] == "int8":
        whole, scale = _to_int8(w, 1)
        state["weights"], state["scales"] = whole.to(torch.int8), scale
    else:
        state["weights"] = w.to(BF16)
    return state


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"product": _own_product, "lowrank": _own_lowrank, "grouped": _own_grouped}[kind](state)
    return {"product": _plain_product, "lowrank": _plain_lowrank, "grouped": _plain_grouped}[kind](state)


def _own_product(s):
    from burn_dragon_amd.packed import product

    return product(s["x"], s["weights"], out_dtype=TYPES[s["case"]["out"]])


def _own_lowrank(s):
    from burn_dragon_amd.kernel.relu_lowrank import packed_forward

    return packed_forward(s["x"], s["weights"], threshold=0.0, gate=s.get("gate"), out_dtype=TYPES[s["case"]["out"]])


def _own_grouped(s):
    from burn_dragon_amd.packed import grouped_product

    return grouped_product(s["x"], s["weights"], s["offsets"], out=s["out"])


def _plain_rows(s):
    """The rows as the product takes them, in 32 bits, and their scales (1 where there are none)."""
    x = s["x"].to(F32)
    return _to_int8(x, -1) if s["case"]["weights"] == "int8" else (x.to(BF16).to(F32), 1.0)


def _plain_product(s):
    rows, scale = _plain_rows(s)
    out = rows @ s["weights"][0].to(F32)
    if "scales" in s:
        out = out * scale * s["scales"][0]
    return out.to(TYPES[s["case"]["out"]])


def _plain_lowrank(s):
    rows, scale = _plain_rows(s)
    B, h_in, T, d = rows.shape
    w = s["weights"].to(F32)
    h, N = w.shape[0], w.shape[2]
    if h_in == 1:
        out = (rows.reshape(B * T, d) @ w.permute(1, 0, 2).reshape(d, h * N)).reshape(B, T, h, N).permute(0, 2, 1, 3)
    else:
        by_head = rows.permute(1, 0, 2, 3).reshape(h, B * T, d).contiguous()
        out = torch.matmul(by_head, w).reshape(h, B, T, N).permute(1, 0, 2, 3)
    if "scales" in s:
        out = out * scale * s["scales"]
    out = torch.where(out > 0, out, torch.zeros((), device=DEVICE))
    if "gate" in s:
        out = out * s["gate"].to(F32)
    return out.contiguous().to(TYPES[s["case"]["out"]])


def _plain_grouped(s):
    """Groups padded to the longest: one product of a batch."""
    rows, scale = _plain_rows(s)
    offsets, most = s["offsets"].to(torch.int64), s["longest"]
    M, G = rows.shape[0], s["weights"].shape[0]
    m = torch.arange(M, device=DEVICE)
    group = (torch.searchsorted(offsets, m, right=True) - 1).clamp(0, G - 1)
    inside = (m >= offsets[0]) & (m < offsets[-1])
    taken = (offsets[:-1, None] + torch.arange(most, device=DEVICE)).clamp(max=M - 1)  # rows past a group's end are not used
    padded = torch.matmul(rows[taken], s["weights"].to(F32))
    out = padded.reshape(G * most, -1)[(group * most + m - offsets[group]).clamp(0, G * most - 1)]
    if "scales" in s:
        out = out * scale * s["scales"][group, 0]
    s["out"].copy_(torch.where(inside[:, None], out.to(s["out"].dtype), s["out"]))
    return s["out"]


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    G, K, N = _dense(case)
    size = {"f32": 4, "bf16": 2, "int8": 1}
    held = K * N * size[case["weights"]] + (4 * N if case["weights"] == "int8" else 0)
    if case["kind"] == "product":
        rows_in = rows_out = case["rows"]
        used = 1.0
    elif case["kind"] == "lowrank":
        rows_out = case["batch"] * case["tokens"] * case["heads"]
        rows_in = case["batch"] * case["tokens"] if case["shared"] else rows_out
        used = float(G)
    else:
        rows_in = rows_out = case["rows"] - min(case["spare"], case["rows"] - 1)
        share = [(g + 1.0) ** -case["skew"] for g in range(G)]
        used = sum(1.0 - (1.0 - p / sum(share)) ** rows_in for p in share)  # groups that get a row
    gate = rows_out * N * size[case["x"]] if case.get("gated") else 0
    return {"bytes": int(rows_in * K * size[case["x"]] + used * held + gate + rows_out * N * size[case["out"]]),
            "flops": int(2 * rows_out * K * N)}


# ---- the definitions in 64 bits ---------------------------------------------------------

def _whole(v, dim):
    """Whole numbers in 64 bits and the scales: a quotient or product of two numbers of 32 bits, made in 64 and rounded to 32,
    is the one that is rounded once."""
    v = v.to(torch.float64)
    top = torch.amax(torch.abs(v), dim, True)
    some = top >= 2.0 ** -118
    top = torch.where(some, top, 1.0)
    up, scale = (127.0 / top).to(F32).to(torch.float64), (top / 127.0).to(F32).to(torch.float64)
    near = torch.round((v * up).to(F32).to(torch.float64))
    return torch.where(some, near, 0.0), torch.where(some, scale, 0.0)


def exact(case, seed):
    """Group by group, in pieces of the outer dimension."""
    state, w = _prepared(case, seed)
    int8 = case["weights"] == "int8"
    x = state["x"]
    if case["kind"] == "lowrank":
        B, T, h = case["batch"], case["tokens"], case["heads"]
        out = torch.empty((B, h, T, case["latent"]), device=DEVICE, dtype=torch.float64)
    else:
        out = torch.zeros((case["rows"], case["outer"]), device=DEVICE, dtype=torch.float64)
    limits = state["offsets"].tolist() if "offsets" in state else None
    for g in range(w.shape[0]):
        if case["kind"] == "lowrank":
            mine = x[:, 0 if case["shared"] else g].reshape(B * T, -1)
        elif limits is None:
            mine = x
        else:
            mine = x[limits[g]:limits[g + 1]]
        if mine.shape[0] == 0:
            continue
        if int8:
            a, sa = _whole(mine, 1)
        else:
            a, sa = mine.to(BF16).to(torch.float64), None
        for n in range(0, w.shape[2], 8192):
            if int8:
                b, sb = _whole(w[g, :, n:n + 8192], 0)
                part = torch.mm(a, b) * (sa * sb)
            else:
                part = torch.mm(a, w[g, :, n:n + 8192].to(BF16).to(torch.float64))
            if case["kind"] == "lowrank":
                part = part.clamp(min=0).reshape(B, T, -1)
                if "gate" in state:
                    part = part * state["gate"][:, g, :, n:n + 8192].to(torch.float64)
                out[:, g, :, n:n + 8192] = part
            elif limits is None:
                out[:, n:n + 8192] = part
            else:
                out[limits[g]:limits[g + 1], n:n + 8192] = part
    return out
