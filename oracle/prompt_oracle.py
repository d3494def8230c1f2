"""CPU oracle of attention over packed prompts, in 64 bits.  TEST INFRASTRUCTURE ONLY: the
product package never imports it."""
from __future__ import annotations

import math

import torch


def attend(q, k, v, scale, softcap=None):
    """q [n, heads, hd], k, v [m, kv_heads, hd]: row i attends rows 0 .. m - n + i of k.  Values
    that a row does not attend have no part in it, whatever they are."""
    n, heads, hd = q.shape
    m, kvh = k.shape[:2]
    out = torch.zeros(n, heads, v.shape[-1], dtype=torch.float64)
    if m == 0:
        return out
    unseen = torch.ones(n, m, dtype=torch.bool).triu(m - n + 1)
    for h in range(heads):
        kk, vv = k[:, h * kvh // heads].double(), v[:, h * kvh // heads].double()
        w = q[:, h].double() @ kk.T * scale
        if softcap:
            w = softcap * torch.tanh(w / softcap)
        w = w.masked_fill(unseen, -math.inf)
        p = torch.softmax(w, dim=-1).masked_fill(unseen, 0.0)
        if torch.isfinite(vv).all():
            o = p @ vv
        else:  # products of the attended positions alone
            o = torch.stack([(p[i, :m - n + i + 1, None] * vv[:m - n + i + 1]).sum(0) if m - n + i >= 0 else
                             torch.zeros(hd, dtype=torch.float64) for i in range(n)])
        out[:, h] = torch.where((~unseen).any(-1)[:, None], o, torch.zeros((), dtype=torch.float64))
    return out


def tolerance(q, k, v, scale, probability_eps, out_eps, want):
    """How far attention in 32 bits may be from 64: probabilities rounded to `probability_eps`,
    scores as sums of hd products in 32 bits (a relative 2^-23 of the sum of magnitudes for each
    addition), an exponential good to 2^-21, sums over the positions in 32 bits, the result
    rounded to `out_eps`."""
    if k.shape[0] == 0:
        return torch.zeros_like(want) + 1e-30
    top = float((q.double().norm(dim=-1).amax() * k.double().norm(dim=-1).amax())) * abs(scale)
    score = top * (q.shape[-1] + 8) * 2.0 ** -23
    e = probability_eps + 2 * (score + 2.0 ** -21) + (math.sqrt(k.shape[0]) + 8) * 2.0 ** -23
    return want.abs() * out_eps + v.double().abs().amax() * e + 1e-30


def packed(q, k, v, cu, cu_k, scale, softcap=None, probability_eps=0.0, out_eps=0.0):
    """(output, tolerance) of packed sequences, zero rows where there is no sequence."""
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[-1], dtype=torch.float64)
    room = torch.full_like(out, 1e-30)
    for b in range(len(cu) - 1):
        a, c = slice(int(cu[b]), int(cu[b + 1])), slice(int(cu_k[b]), int(cu_k[b + 1]))
        out[a] = attend(q[a], k[c], v[c], scale, softcap)
        if a.stop > a.start:
            room[a] = tolerance(q[a], k[c], v[c], scale, probability_eps, out_eps, out[a])
    return out, room
