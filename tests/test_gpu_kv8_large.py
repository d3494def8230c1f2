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


@pytest.mark.parametrize("io,hd,heads,kvh,bs,sl,at_once", [
    (BF, 128, 48, 8, 4, 2048, 16), (BF, 128, 40, 4, 2, 5000, 32), (HF, 128, 42, 2, 2, 4096, 16), (F32, 128, 12, 2, 4, 2500, 8),
    (HF, 64, 12, 4, 8, 2500, 8), (BF, 64, 36, 2, 5, 4001, 32)])
@pytest.mark.parametrize("norm,halves", [(False, True), (True, False)])
def test_queries_of_large_prompts(io, hd, heads, kvh, bs, sl, at_once, norm, halves):
    """A lane takes 8, 16 or 32 heads of its position, the last group partly full."""
    A = base._attention()
    gen = torch.Generator(device="cuda").manual_seed(heads + sl)
    cpu = torch.Generator().manual_seed(heads)
    # the rule of the launch
    want, groups = torch.cuda.get_device_properties(0).multi_processor_count * 8 * (256 // (hd // 8)), 4
    while groups < heads and bs * sl * ((heads - 1) // (2 * groups) + 1) >= want:
        groups *= 2
    assert groups == at_once
    cache = base._cache(io, kvh, hd, 32, layers=1)
    per = -(-(sl + 9 * bs) // 32)
    ids = torch.randperm(bs * per, generator=cpu).view(bs, per).to(torch.int32).cuda()
    state = cache.allocate(bs * per)
    w = base.Write(cache, heads, io, cpu, norm, halves)
    q, k, v = (torch.randn(bs, sl, n, hd, generator=gen, device="cuda").to(io) for n in (heads, kvh, kvh))
    start = torch.arange(bs) * 9
    got = w.call(state, ids, start, q, k, v, layer=0)
    assert base._status() == 0
    slab = state[0].unflatten(1, cache.sub_page_dims)
    for b in range(bs):
        at = torch.cat([torch.randint(0, sl, (60,), generator=cpu), torch.tensor([0, 1, 31, 32, sl - 2, sl - 1])])
        qb, kb, vb = (t[b, at.cuda()].cpu() for t in (q, k, v))
        pos = int(start[b]) + at
        for x, g, wt in ((qb, got[0], w.w[0]), (kb, got[1], w.w[1])):
            y = ko.turn(x, pos, w.freqs, wt, halves=halves)
            size = x.double().abs().amax(-1, keepdim=True)
            if wt is not None:
                size = size * wt.abs().max() / x.double().pow(2).mean(-1, keepdim=True).add(1e-5).sqrt()
            d = size * 16 * 2.0 ** -23
            off = (g[b, at.cuda()].cpu().double() - y).abs() - d - base.EPS[io] * (y.abs() + d) - base.FLOOR[io]
            assert off.max() <= 0, float(off.max())
        page = ids[b, (pos // 32).cuda()].long()
        held = slab[page, 0, :, (pos % 32).cuda()]
        assert torch.equal(held[:, 0], got[1][b, at.cuda()]) and torch.equal(held[:, 1].cpu(), vb)


@pytest.mark.parametrize("code", [I8, BF])
def test_more_than_65535_ctas_of_keys_and_values(code):
    """K and V of many short rows: their CTAs are found among the others in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(17)
    bs, heads, kvh, hd = 33_333, 4, 2, 64
    cache = base._cache(code, kvh, hd, 4, layers=1)
    state = cache.allocate(bs)
    ids = torch.randperm(bs, generator=torch.Generator().manual_seed(18)).to(torch.int32)[:, None].cuda()
    w = base.Write(cache, heads, BF, None)
    q, k, v = (torch.randn(bs, 1, n, hd, generator=gen, device="cuda").to(BF) for n in (heads, kvh, kvh))
    start = torch.arange(bs) % 4
    got = w.call(state, ids, start, q, k, v, layer=0)
    assert base._status() == 0
    turned = [ko.turn(x.cpu(), start[:, None], w.freqs) for x in (q, k)]
    for x, y, g in zip((q, k), turned, got):
        d = x.cpu().double().abs().amax(-1, keepdim=True) * 16 * 2.0 ** -23
        off = (g.cpu().double() - y).abs() - d - base.EPS[BF] * (y.abs() + d)
        assert off.max() <= 0, float(off.max())
    page, seq = ids[:, 0].long().cpu(), torch.arange(bs)
    if code == BF:
        held = state[0].unflatten(1, cache.sub_page_dims).cpu()
        for slot, x in enumerate((got[1], v)):
            assert torch.equal(held[page, 0, slot, start], x[:, 0].cpu())
        held[page, 0, :, start] = 0
        assert not held.any()
        return
    codes, scales = ko.page_views(state, cache)  # blocks of four positions; a fresh page's scale is 0
    s, c = scales[page, 0, :, 0], codes[page, 0, :, :, start]
    for slot, x in enumerate((turned[1][:, 0], v[:, 0].cpu().double())):
        amax = x.abs().amax(-1)
        assert ((s[..., slot] * 127 - amax).abs() <= amax * 2.0 ** -18).all()
        y = x / s[..., slot, None]
        assert ((c[:, :, slot] - y).abs() <= 0.5 * (1 + 2.0 ** -10) + 127 * 2.0 ** -18).all()
