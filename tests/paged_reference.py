"""The paged-serving operators from their definitions, in 64 bits (torch, any device), for the tests."""
import math

import torch

# Largest relative rounding of each type: half a step.
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rotate(x, cos, sin):
    """x f64 [n, heads, Dh], cos / sin f64 [n, half] of the rows' positions."""
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def quantise(x):
    """f32 rows [.., Dh] -> codes [.., Dh] (0..15) and f16 scales [.., Dh / 32], by comparing with every level's border."""
    blocks = x.double().unflatten(-1, (-1, 32))
    big = blocks.abs().amax(-1, keepdim=True)
    first = (blocks.abs() == big).to(torch.int8).argmax(-1, keepdim=True)
    d = (blocks.gather(-1, first) / -8).clamp(-65504, 65504).float().half()
    df = d.double()
    borders = (torch.arange(1, 16, dtype=torch.float64, device=x.device) - 8.5) * df.abs()[..., None]
    code = ((blocks * torch.sign(df))[..., None] >= borders).sum(-1)
    code = torch.where(df == 0, torch.full_like(code, 8), code)
    return code.flatten(-2).to(torch.uint8), d.squeeze(-1)


def key_nibble(Dh):
    """Nibble of a key row that holds dimension i."""
    nb = Dh // 32
    return torch.tensor([((i % 32 // 8) * nb + i // 32) * 8 + i % 8 for i in range(Dh)])


def value_nibble(Dh):
    nb = Dh // 32
    return torch.tensor([((i % 32 // 4) * nb + i // 32) * 4 + i % 4 for i in range(Dh)])


def pack(code, order):
    """Codes [.., Dh] -> bytes [.., Dh / 2] with dimension i in nibble order[i]."""
    nib = torch.empty_like(code)
    nib[..., order.to(code.device)] = code
    nib = nib.unflatten(-1, (-1, 2))
    return nib[..., 0] | (nib[..., 1] << 4)


def unpack(rows, scale, order):
    """Bytes [.., Dh / 2] and scales [.., Dh / 32] -> f64 values [.., Dh]."""
    nib = torch.stack([rows & 15, rows >> 4], -1).flatten(-2)
    code = nib[..., order.to(rows.device)].double() - 8
    return code * scale.double().repeat_interleave(32, -1)


def cache_rows(cache, slots, which):
    """f64 values [n, KV, Dh] of the cache rows that slots name."""
    page, off = slots // cache.page_size, slots % cache.page_size
    rows, scale = (cache.k, cache.k_scale) if which == "k" else (cache.v, cache.v_scale)
    order = key_nibble(cache.head_dim) if which == "k" else value_nibble(cache.head_dim)
    return unpack(rows[page, :, off], scale[page, :, off], order)


def attend(q, k, v, first, window=0, missing=None):
    """q f64 [S, H, D] at positions first .. over k, v f64 [T, KV, D].  Returns the output and, for error bounds,
    sum_j p_j |v_j| per element and the largest sum_d |q_d k_jd| / sqrt(D) per (query, head) over its visible keys.
    `missing`: bool [T], tokens that are left out."""
    S, H, D = q.shape
    T, KV, _ = k.shape
    G = H // KV
    pos = first + torch.arange(S, device=q.device)[:, None]
    t = torch.arange(T, device=q.device)[None]
    see = t <= pos
    if window:
        see = see & (t > pos - window)
    if missing is not None:
        see = see & ~missing[None]
    kh, vh = (x.repeat_interleave(G, 1).transpose(0, 1) for x in (k, v))  # [H, T, D]
    x = torch.matmul(q.transpose(0, 1), kh.transpose(1, 2)) / math.sqrt(D)  # [H, S, T]
    mag = torch.matmul(q.abs().transpose(0, 1), kh.abs().transpose(1, 2)) / math.sqrt(D)
    x = torch.where(see[None], x, -math.inf)
    p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
    out = torch.matmul(p, vh).transpose(0, 1)
    spread = torch.matmul(p, vh.abs()).transpose(0, 1)
    mag = torch.where(see[None], mag, 0.0).amax(-1).transpose(0, 1) if T else torch.zeros((S, H), dtype=torch.float64, device=q.device)
    return out, spread, mag


def attention_bound(out, spread, mag, D, T, dtype, p_half_step=2.0 ** -22, v_max=None):
    """What f32 arithmetic can be off by.  A score is a sum of D products: its error is at most (D + 8) steps of 2^-24 of
    sum |q k| (the products' and the sum's roundings, the scale and the exponent's argument), which moves each probability by
    that factor and its normalisation by as much; the exponential and the division add a few steps, the probabilities'
    own rounding p_half_step, and the sum over T tokens T / 16 + 16 steps (it runs 16 tokens at a time); the result is
    rounded once."""
    u = 2.0 ** -24
    rel = 2 * (D + 8) * u * mag[..., None] + 16 * u + p_half_step * 1.01 + (T / 16 + 32) * u
    return rel * spread + HALF_STEP[dtype] * 1.01 * out.abs() + 1e-30
