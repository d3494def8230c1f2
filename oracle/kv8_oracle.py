"""CPU oracle of the 8-bit KV cache, in 64 bits.  TEST INFRASTRUCTURE ONLY: the product
package never imports it.

Definitions: a scale block is `block` consecutive positions of a page; a code c of the
block, head and K | V with scale s stands for c * s.  There is no counterpart in the
reference beyond its per-tensor quantizer; the rotation and the norm are those of
attention_oracle.py.
"""
from __future__ import annotations

import math

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FITS = 1.0 + 2.0 ** -10   # how far above qmax a value still rounds to it
ZERO = 2.0 ** -100        # scales below count as zero


def turn(x, pos, freqs, weight=None, eps=1e-5, halves=False):
    """Norm and rotation of x [..., heads, hd] at pos [...], in 64 bits."""
    x = x.double()
    if weight is not None:
        x = weight.double() * x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    a = (pos.double()[..., None] * freqs.double())[..., None, :]
    c, s = torch.cos(a), torch.sin(a)
    out = torch.empty_like(x)
    if halves:
        h = x.shape[-1] // 2
        out[..., :h] = x[..., :h] * c - x[..., h:] * s
        out[..., h:] = x[..., h:] * c + x[..., :h] * s
    else:
        out[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
        out[..., 1::2] = x[..., 1::2] * c + x[..., 0::2] * s
    return out


def half_step(y, dtype):
    """Half the distance of the codes around y (in units of the scale), 64 bits."""
    if dtype == torch.int8:
        return torch.full_like(y, 0.5)
    return torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 4)


def to_code(y, dtype):
    """Nearest code, ties to even, as a 64-bit number."""
    y = y.clamp(-QMAX[dtype], QMAX[dtype])
    step = 2 * half_step(y, dtype)
    return torch.round(y / step) * step


def page_views(state, cache):
    """codes [pages, blocks, heads, 2, stride, hd] and scales [pages, blocks, heads, n, 2] as 64-bit copies."""
    codes = state[0].cpu().view(torch.int8).view(cache.dtype).to(torch.float32).double().unflatten(1, cache.sub_page_dims)
    return codes, state[1].cpu().double().unflatten(1, cache.scale_page_dims)


def growth(amax: float, scale: float, qmax: float) -> int:
    """By how many powers of two a continued block's scale grows."""
    k = 0
    while amax > scale * 2.0 ** k * qmax * FITS:
        k += 1
    return k


def gather(codes, scales, cache, layer, ids, n):
    """Values of the first n positions of one sequence: [2, n, heads, hd]."""
    out = torch.zeros(2, n, cache.attn_head_count, cache.attn_head_dim, dtype=torch.float64)
    for p in range(n):
        page, off = int(ids[p // cache.block_seq_stride]), p % cache.block_seq_stride
        s = scales[page, layer, :, off // cache.scale_block]          # [heads, 2]
        out[:, p] = (codes[page, layer, :, :, off] * s[..., None]).transpose(0, 1)
    return out


def attend(q, k, v, lens_visible, scale, softcap=None):
    """q [sl, heads, hd], k, v [n, kv_heads, hd]; token i sees the first lens_visible[i] positions."""
    sl, heads, hd = q.shape
    rep = heads // k.shape[1]
    k, v = k.repeat_interleave(rep, dim=1), v.repeat_interleave(rep, dim=1)
    out = torch.zeros(sl, heads, hd, dtype=torch.float64)
    for i in range(sl):
        n = lens_visible[i]
        if n <= 0:
            continue
        w = torch.einsum("hd,nhd->hn", q[i].double(), k[:n]) * scale
        if softcap:
            w = softcap * torch.tanh(w / softcap)
        out[i] = torch.einsum("hn,nhd->hd", torch.softmax(w, dim=-1), v[:n])
    return out


def attend_tolerance(q, k, v, scale, probability_eps, out_eps, want):
    """How far attention in 32 bits may be from 64: rounding of the probabilities to
    `probability_eps`, scores as sums of hd products in 32 bits (a relative 2^-23 of the sum
    of magnitudes for each addition), an exponential good to 2^-21, sums over the positions
    in 32 bits, the result rounded to `out_eps`."""
    if k.shape[0] == 0:
        return torch.zeros_like(want) + 1e-30
    rep = q.shape[1] // k.shape[1]
    kk = k.abs().repeat_interleave(rep, dim=1)
    top = torch.einsum("shd,nhd->shn", q.double().abs(), kk).amax() * abs(scale)
    score = float(top) * (q.shape[-1] + 8) * 2.0 ** -23
    e = probability_eps + 2 * (score + 2.0 ** -21) + (math.sqrt(k.shape[0]) + 8) * 2.0 ** -23
    return want.abs() * out_eps + v.abs().amax() * e + 1e-30
