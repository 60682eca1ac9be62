"""A model whose projections are packed, in 64 bits: the layer of oracle/bdh_oracle.py with rows and weights rounded to 8 bits or
bf16 where the packed products round them."""
import numpy as np
import torch

from oracle import bdh_oracle as orc


def whole(v, axis, near):
    """Whole numbers and scales.  Of the weights (near is None) by the rule in 32 bits; of rows, whose device values differ by
    roundings, in 64 bits: the least distance of a quotient from a border between two whole numbers goes into `near`."""
    v = v.astype(np.float32 if near is None else np.float64)
    of = v.dtype.type
    top = np.abs(v).max(axis=axis, keepdims=True)
    fits = top >= of(2.0**-118)
    safe = np.where(fits, top, of(1.0))
    z = v * (of(127.0) / safe)
    if near is not None:
        near.append(np.abs(np.abs(z - np.floor(z)) - 0.5)[np.broadcast_to(fits, z.shape)].min(initial=0.5))
    return np.where(fits, np.rint(z), 0.0).astype(np.float64), np.where(fits, safe / of(127.0), 0.0).astype(np.float64)


def bf16(v, near):
    r = torch.from_numpy(np.ascontiguousarray(v)).to(torch.float32).to(torch.bfloat16).double().numpy()
    if near is not None:  # distance from the middle between two bf16 numbers, in steps
        with np.errstate(divide="ignore"):
            step = np.exp2(np.floor(np.log2(np.abs(v))) - 7)
        off = np.where(v == 0, 0.0, np.abs(v - r) / np.where(step == 0, 1.0, step))
        near.append((0.5 - off).min(initial=0.5))
    return r


def product(x, w, kind, near=None):
    """x [..., K] times w [K, N] (or [..., K, N])."""
    if kind is torch.int8:
        (q, s), (p, t) = whole(x, -1, near), whole(w, -2, None)
        return np.matmul(q, p) * s * t
    return np.matmul(bf16(x, near), bf16(w, None))


def forward_with_state(shape, w, tokens, state, kind, near):
    """orc.forward_with_state with packed projections."""
    B, T = tokens.shape
    h, d, N = shape.n_head, shape.n_embd, shape.latent_per_head
    Nq = 2 * N if shape.rotary == orc.POPE else N
    cur = orc.layer_norm(w.embed[tokens].reshape(B, 1, T, d))
    freqs = orc.build_freqs(N, shape.rope_theta, shape.rotary, np.float32).astype(np.float64)
    decay = orc.alibi_decay(orc.default_alibi_slopes(h, np.float64)) if shape.rotary == orc.ALIBI else None
    for layer in range(shape.n_layer):
        x = np.maximum(product(cur, w.encoder, kind, near) - shape.relu_threshold, 0.0)
        rho = state.rho[layer]
        rho = np.zeros((B, h, Nq, d)) if rho is None else rho
        attn, state.rho[layer] = orc.recurrent_attention(orc.rotate(x, freqs, shape.rotary, state.position), cur[:, 0], rho, decay)
        y = np.maximum(product(orc.layer_norm(attn), w.encoder_v, kind, near) - shape.relu_threshold, 0.0)
        mixed = np.swapaxes(x * y, 1, 2).reshape(B * T, h * N)
        cur = orc.layer_norm(cur + orc.layer_norm(product(mixed, w.decoder, kind, near).reshape(B, 1, T, d)))
    state.position += T
    return np.matmul(cur.reshape(B * T, d), w.lm_head).reshape(B, T, shape.vocab_size)
