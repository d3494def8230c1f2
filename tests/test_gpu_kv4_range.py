"""The operators of the 4-bit KV cache at the ends of their range, against their definition
in 64 bits."""
import math

import pytest
import torch

import test_gpu_kv4 as base
from oracle import kv4_oracle as k4, prompt_oracle as po

pytestmark = pytest.mark.gpu

BF, HF, F32, EPS = base.BF, base.HF, base.F32, base.EPS


def _attend(cache, state, ids, n, q, **kw):
    return base._attention().kv_attend(q.cuda(), cache, state, block_index=0, seq_block_ids=ids.cuda(),
                                       seq_lens=torch.tensor([n]).cuda(), **kw).cpu()


def _check(got, q, k, v, terms, out_dtype, p_eps, softcap=None, norm=True):
    """terms: the largest sum of magnitudes of a position's terms of a score, from the scales and
    offsets of K.  Scores are sums of hd + 16 roundings of 2^-23 of it; a weight is off by twice that.
    In the 2-norm as for keys of size one: the roundings are relative."""
    want = po.attend(q, k, v, q.shape[-1] ** -0.5, softcap)
    e = p_eps + 2 * (terms * (q.shape[-1] + 16) * 2.0 ** -23 + 2.0 ** -21) + (math.sqrt(k.shape[0]) + 8) * 2.0 ** -23
    off = (got.double() - want).abs()
    room = want.abs() * EPS[out_dtype] + 3 * v.abs().amax() * e
    assert (off - room).max() <= 0, (float(off.max()), float((off - room).max()))
    if norm:
        most = math.sqrt(3 * p_eps ** 2 + EPS[out_dtype] ** 2) / math.sqrt(3) + 2.0 ** -18
        assert float(off.norm() / want.norm()) <= most, float(off.norm() / want.norm())


@pytest.mark.parametrize("io,out_dtype,softcap", [(F32, F32, None), (F32, BF, None), (BF, F32, None), (BF, BF, 300.0), (HF, HF, None), (BF, BF, None)])
@pytest.mark.parametrize("size", [2.0 ** -15, 2.0 ** -10, 2.0 ** -5, 1.0, 2.0 ** 8, 2.0 ** 12, 2.0 ** 13])
@pytest.mark.parametrize("hd", [64, 128])
def test_keys_of_all_sizes(size, io, out_dtype, softcap, hd):
    """K of one size, queries of its inverse, so that scores are of order one; offsets of either sign."""
    gen = torch.Generator().manual_seed(int(100 + math.log2(size)))
    cache = base._cache(2, hd, 16, layers=1)
    state = k4.fill(cache, 12, gen)
    half = state[1].view(12, 2, 2, 16, hd // 32, 2)
    half[:, :, 0] = (half[:, :, 0].cpu().float() * size).half()
    half[3, :, 0, 5, :, 1] = 0.0                       # groups from zero up
    if size == 2.0 ** 13:                              # m and s in fp16's range, m + 8 s and m + 15 s beyond
        half[4, :, 0, 2] = torch.tensor([4500.0, 30000.0]).half()
        half[5, :, 0, 3, 0] = torch.tensor([9333.0, 0.0]).half()
        half[6, :, 0, 7, 1] = torch.tensor([8.0, 65500.0]).half()
        half[7, :, 0, 7, 1] = torch.tensor([8192.0, -65504.0]).half()
    ids = torch.arange(10, dtype=torch.int32).view(1, 10) + 1
    codes, held = k4.page_views(state, cache)
    assert torch.isfinite(held).all()
    q = (torch.randn(1, 2, 8, hd, generator=gen) / size).clamp(-6e4, 6e4).to(io)
    for n in (150, 37):
        k, v = k4.gather(codes, held, cache, 0, ids[0], n)
        # K's terms: codes less 8 times the scale and the offset 8 scales up, or codes and offset
        mag = (held[ids[0].long(), 0, :, 0, :, :, 0].abs() * 15 + held[ids[0].long(), 0, :, 0, :, :, 1].abs()).amax()
        top = float(q.double().abs().sum(-1).amax() * mag) * hd ** -0.5
        p_eps = 2.0 ** -11 if out_dtype == BF and io != F32 and softcap is None else 2.0 ** -20
        _check(_attend(cache, state, ids, n, q, out_dtype=out_dtype, softcap=softcap)[0], q[0], k, v, top, out_dtype, p_eps, softcap,
               norm=size < 2.0 ** 13)
    assert base._status() == 0


@pytest.mark.parametrize("io", [BF, HF, F32])
@pytest.mark.parametrize("hd,new", [(64, 1), (64, 4), (128, 1), (128, 4)])
@pytest.mark.parametrize("n", [100, 700])
def test_a_bad_group_of_values_shows_in_its_elements(io, hd, new, n):
    """NaN in the scales of some groups of V: NaN in their 32 elements of the rows that see the position,
    the other elements as if the group were zero."""
    gen = torch.Generator().manual_seed(n + hd)
    cache = base._cache(2, hd, 16, layers=1)
    per = -(-n // 16)
    ids = base._ids(1, per, gen)
    state = k4.fill(cache, per + 2, gen)
    half = state[1].view(per + 2, 2, 2, 16, hd // 32, 2)
    q = torch.randn(1, new, 8, hd, generator=gen).to(io)
    places = [(n - 2, 0, 1), (17, 1, 0), (n // 2, 1, hd // 32 - 1), (n - 1, 1, 0)]  # position, kv head, group
    for p, h, g in places:
        half[int(ids[0, p // 16]), h, 1, p % 16, g] = 0.0
    # a group whose scales would not matter beside it
    codes, held = k4.page_views(state, cache)
    k, v = k4.gather(codes, held, cache, 0, ids[0], n)
    for p, h, g in places:
        half[int(ids[0, p // 16]), h, 1, p % 16, g] = math.nan
    got = _attend(cache, state, ids, n, q)
    hit = torch.zeros(new, 8, hd, dtype=torch.bool)
    for p, h, g in places:
        hit[torch.arange(new) + n - new >= p, 4 * h:4 * h + 4, 32 * g:32 * g + 32] = True
    assert torch.equal(torch.isnan(got[0]), hit)
    want = po.attend(q[0], k, v, hd ** -0.5)
    p_eps = 2.0 ** -11 if io == BF else 2.0 ** -20
    top = float(q.double().abs().sum(-1).amax() * held.abs().max() * 16) * hd ** -0.5
    e = p_eps + 2 * (top * (hd + 16) * 2.0 ** -23 + 2.0 ** -21) + (math.sqrt(n) + 8) * 2.0 ** -23
    off = (got[0].double() - want).abs()[~hit]
    assert (off - want.abs()[~hit] * EPS[io] - 3 * 16 * held.abs().max() * e).max() <= 0
    # the read-back agrees on which
    kk, vv = base._attention().kv_read(cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=torch.tensor([n]).cuda(), max_seq_len=n)
    bad = torch.zeros(n, 2, hd, dtype=torch.bool)
    for p, h, g in places:
        bad[p, h, 32 * g:32 * g + 32] = True
    assert torch.equal(torch.isnan(vv[0].cpu()), bad)
    assert base._status() == 0
