"""The operators of the 8-bit KV cache at sizes that take other ways through the kernels:
long lists of attention steps, large prompts, many sequences; against the definition
in 64 bits."""
import pytest
import torch

import test_gpu_kv8 as base
from oracle import kv8_oracle as ko

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("code,io,hd,heads,kvh,sl,bs", [
    (I8, BF, 128, 32, 8, 1, 64), (E4, BF, 64, 16, 8, 1, 90), (I8, F32, 128, 16, 8, 1, 64), (E4, HF, 128, 32, 8, 2, 64),
    (E4, BF, 128, 32, 8, 4, 64), (I8, F32, 64, 24, 8, 3, 90), (I8, BF, 128, 48, 8, 5, 64)])
def test_long_lists_of_steps(code, io, hd, heads, kvh, sl, bs):
    """More than four steps for every CTA, where segments count more steps than they have: ragged
    and empty sequences, whole and split segments."""
    from shark_platform_b200 import _cabi as C
    import ctypes

    A = base._attention()
    gen = torch.Generator().manual_seed(hd + heads + sl)
    cache = base._cache(code, kvh, hd, 32, 16, layers=1)
    pages, per = 60, 36
    state = base._fill(cache, pages, gen)
    # attention only reads: sequences may share pages
    ids = torch.stack([torch.randperm(pages, generator=gen)[:per] for _ in range(bs)]).to(torch.int32)
    lens = torch.randint(0, 1100, (bs,), generator=gen)
    lens[::9] = torch.randint(0, 4, (len(lens[::9]),), generator=gen)
    lens[4], lens[7], lens[-1] = 128, 1151, 129
    q = torch.randn(bs, sl, heads, hd, generator=gen).to(io)
    rows = heads // kvh * sl
    tile = 8 if rows <= 8 else 16
    desc = C.Kv8CacheDesc(1, 32, kvh, hd, pages, 16, C.KV8_INT8 if code == I8 else C.KV8_E4M3)
    ctas = C.lib.b200moe_kv8_attend_scratch_bytes(ctypes.byref(desc), bs, sl, heads, per * 32) // (2 * tile * (hd + 4) * 4)
    steps = int(((lens + 127) // 128).clamp(min=1).sum()) * kvh * -(-rows // tile)
    assert steps >= 4 * ctas, (steps, ctas)
    got = A.kv_attend(q.cuda(), cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=lens.cuda())
    again = A.kv_attend(q.cuda(), cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=lens.cuda())
    assert base._status() == 0 and torch.equal(got, again)
    codes, scales = ko.page_views(state, cache)
    for b in sorted({0, 1, 4, 7, 9, bs - 2, bs - 1, *range(2, bs, 5)}):
        n = int(lens[b])
        k, v = ko.gather(codes, scales, cache, 0, ids[b], n)
        want = ko.attend(q[b], k, v, [n - sl + 1 + i for i in range(sl)], hd ** -0.5)
        room = ko.attend_tolerance(q[b], k, v, hd ** -0.5, 2.0 ** -11 if io != F32 else 2.0 ** -21, base.EPS[io], want) + base.FLOOR[io]
        off = (got[b].cpu().double() - want).abs()
        assert bool((off <= room).all()), (b, n, float((off / room).max()))
