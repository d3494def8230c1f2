"""CPU oracle of the 4-bit KV cache, in 64 bits.  TEST INFRASTRUCTURE ONLY: the product
package never imports it.

Definitions: 32 consecutive values of a row have an fp16 scale s and offset m; a code c,
0 .. 15, stands for c * s + m.  Rotation, norm and attention are kv8_oracle.py's.
"""
from __future__ import annotations

import torch

GROUP = 32


def groups(x):
    """[..., hd] -> [..., hd / 32, 32]"""
    return x.unflatten(-1, (-1, GROUP))


def scales_of(x):
    """(s, m) of rows x [..., hd], fp16 numbers in 64 bits: the difference, the division by 15 and the
    rounding to fp16 as 32-bit arithmetic has them."""
    y = groups(x.float())
    lo, hi = y.amin(-1), y.amax(-1)
    return torch.stack([((hi - lo) / 15.0).half(), lo.half()], dim=-1).double()


def quotients(x, held):
    """(x - m) / s in 64 bits, 0 where s is; held [..., hd / 32, 2]."""
    s, m = held[..., :1], held[..., 1:]
    return torch.where(s > 0, (groups(x.double()) - m) / s, torch.zeros((), dtype=torch.float64)).flatten(-2)


def to_code(y):
    """Nearest code, ties to even."""
    return torch.round(y.clamp(0, 15))


def values(codes, held):
    return (groups(codes.double()) * held[..., :1] + held[..., 1:]).flatten(-2)


def pack(codes):
    c = codes.to(torch.uint8)
    return c[..., 0::2] | c[..., 1::2] << 4


def page_views(state, cache):
    """codes [pages, blocks, heads, 2, stride, hd] and (s, m) [pages, blocks, heads, 2, stride, hd / 32, 2] as 64-bit copies."""
    b = state[0].cpu().unflatten(1, cache.sub_page_dims)
    codes = torch.stack([b & 15, b >> 4], dim=-1).flatten(-2).double()
    return codes, state[1].cpu().double().unflatten(1, cache.scale_page_dims)


def fill(cache, pages, gen, std=1.5):
    """Pages that hold quantised normal values everywhere."""
    state = cache.allocate(pages)
    dims = cache.sub_page_dims[:-1] + [cache.attn_head_dim]
    x = torch.randn(pages, *dims, generator=gen) * std
    held = scales_of(x)
    state[0].copy_(pack(to_code(quotients(x, held))).flatten(1))
    state[1].copy_(held.half().flatten(1))
    return state


def gather(codes, held, cache, layer, ids, n):
    """Values of the first n positions of one sequence: [2, n, heads, hd]."""
    p = torch.arange(n)
    page, off = ids.long()[p // cache.block_seq_stride], p % cache.block_seq_stride
    return values(codes[page, layer, :, :, off], held[page, layer, :, :, off]).permute(2, 0, 1, 3)
