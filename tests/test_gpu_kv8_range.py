"""The operators of the 8-bit KV cache at the ends of their range, against their definition
in 64 bits."""
import pytest
import torch

import test_gpu_kv8 as base
from oracle import kv8_oracle as ko

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io", [BF, F32])
@pytest.mark.parametrize("small,large", [(-88, 38), (-88, 39), (-88, 41), (-80, 50), (-88, 100), (-20, 107), (-20, 110)])
def test_a_block_that_grows_by_any_power_of_two(code, io, small, large):
    """Rows of size 2^small, then one of 2^large behind them in the same block: the quotient of
    the two does not fit 32 bits where they are 2^128 apart."""
    A = base._attention()
    gen = torch.Generator().manual_seed(small - large)
    cache = base._cache(code, 2, 64, 16, 16, layers=1)
    state = cache.allocate(2)
    ids = torch.tensor([[1]], dtype=torch.int32)
    rows = [(torch.randn(1, n, 2, 64, generator=gen) * 2.0 ** size).to(io) for n, size in ((3, small), (1, large))]
    kw = dict(block_index=0, seq_block_ids=ids.cuda(), freqs=base._freqs(64).cuda())
    scales = []
    for x, start in zip(rows, (0, 3)):
        A.norm_rope_kv_write(x.cuda(), x.cuda(), x.cuda(), cache, state, start_positions=torch.tensor([start]).cuda(), **kw)
        scales.append(ko.page_views(state, cache)[1][1, 0, :, 0])
    codes = ko.page_views(state, cache)[0][1, 0]
    assert base._status() == 0
    qmax = ko.QMAX[code]
    turned = [ko.turn(x, torch.arange(s, s + x.shape[1])[None], base._freqs(64)) for x, s in zip(rows, (0, 3))]
    for h in range(2):
        for slot, (first, new) in enumerate((turned, [x.double() for x in rows])):
            new = new[0, 0, h]
            old, s = float(scales[0][h, slot]), float(scales[1][h, slot])
            # the rotation's error is at most 2^-19 of the largest value: nowhere near a border here
            grow = ko.growth(float(new.abs().max()), old, qmax)
            assert s == old * 2.0 ** grow
            y = new / s
            room = ko.half_step(y, code) * (1 + 2.0 ** -10) + y.abs().max() * 2.0 ** -18
            assert ((codes[h, slot, 3] - y).abs() - room <= 0).all()
            # what the earlier rows come to in steps of the new scale: the code they had, and its rounding
            y = first[0, :, h] / s
            assert ((codes[h, slot, :3] - y).abs() <= ko.half_step(y, code) * 2 + y.abs().max() * 2.0 ** -4).all()


@pytest.mark.parametrize("io", [HF, BF])
@pytest.mark.parametrize("hd,halves,stretch", [(128, False, 1.0), (64, True, 1.0), (64, False, 40.0)])
@pytest.mark.parametrize("start", [0, 8000, 130_000, 1_047_000, 6_000_000, (1 << 24) - 2048, (1 << 30) + 12345])
def test_angles_of_16_bit_rows(io, hd, halves, stretch, start):
    """Rows are the 64-bit rotation rounded once, at any position and for frequencies above
    one.  A value is re * cos - im * sin: with cosine and sine good to 2^-20, the angle's part of
    its error is at most (|re| + |im|) 2^-20, and the product and the sum in 32 bits add 2^-24
    of as much each.  Angles of many turns: the products of the definition and of the kernel in
    64 bits are rounded by 2^-53 of the angle, four times in all."""
    A = base._attention()
    gen = torch.Generator().manual_seed(start % 1000)
    cache = base._cache(BF, 1, hd, 32, layers=1)
    sl, heads = 4096, 1024 // hd
    q = (torch.rand(1, sl, heads, hd, generator=gen) * 2 - 1).to(io).cuda()
    k = q[:, :, :1].contiguous()
    freqs = (base._freqs(hd) * stretch).cuda()
    got = A.norm_rope_kv_write(q, k, k, cache, cache.allocate(1), block_index=0, freqs=freqs, use_hf=halves,
                               seq_block_ids=torch.zeros(1, 1, dtype=torch.int32).cuda(),
                               start_positions=torch.tensor([start]).cuda(), new_lens=torch.tensor([0]).cuda())
    assert base._status() == 0
    pos = start + torch.arange(sl, device="cuda")[None]
    for x, y in zip((q, k), got):
        want = ko.turn(x, pos, freqs, halves=halves)
        pair = x.double().abs().unflatten(-1, (2, hd // 2) if halves else (hd // 2, 2))
        at = -2 if halves else -1
        size = pair.sum(at, keepdim=True).expand_as(pair).flatten(-2)
        half = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -14))) - (11 if io == HF else 8))
        angle = (start + sl) * float(freqs.max())
        over = (y.double() - want).abs() - half - size * (2.0 ** -20 + 2 * 2.0 ** -24 + angle * 2.0 ** -51)
        assert over.max() <= 0, float(over.max())


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io", [BF, HF, F32])
def test_values_halfway_between_two_codes(code, io):
    """V whose quotient by amax / qmax is exactly between two codes takes the even one.  16-bit
    activations meet them often: half of the largest value is 63.5 steps of an int8 block."""
    A = base._attention()
    qmax = ko.QMAX[code]
    rows = []
    for m in range(1, 37):
        if code == I8:  # v / amax * 127 = odd / 2: half of amax; of 127 / 64 also others
            for top in range(64 + m, 128, 36):
                rows.append([top / 64.0, top / 128.0, -top / 128.0] + ([j / 128.0 for j in range(1, 122, 2)] if top == 127 else []))
        elif 7 * m < 256:  # v / amax * 448 with an odd five-bit number before the last place: odd * m of amax = 7 m
            rows.append([7.0 * m] + [odd * m * 2.0 ** -e for odd in range(17, 32, 2) if odd * m < 256
                                     for e in range(3, 9) if odd * m * 2.0 ** -e <= 7 * m])
    v = torch.zeros(len(rows), 64)
    for i, r in enumerate(rows):
        v[i, :min(len(r), 64)] = torch.tensor(r[:64])
    v = v.to(io)
    n = len(rows)
    cache = base._cache(code, 1, 64, 1, 1, layers=1)  # a block for each row
    state = cache.allocate(n)
    x = v[None, :, None].cuda()
    A.norm_rope_kv_write(x, x, x, cache, state, block_index=0, seq_block_ids=torch.arange(n)[None].cuda(),
                         start_positions=torch.tensor([0]).cuda(), freqs=base._freqs(64).cuda())
    assert base._status() == 0
    codes = ko.page_views(state, cache)[0][:, 0, 0, 1, 0]
    amax = v.double().abs().amax(-1, keepdim=True)
    y = v.double() * qmax / amax  # exact where it lies between two codes
    step = 2 * ko.half_step(y, code)
    tie = (y / step * 2) % 2 == 1
    assert int(tie.sum()) >= (100 if code == I8 else 300)
    assert torch.equal(codes, ko.to_code(y, code))


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io,hd,heads,kvh,sl,softcap", [(HF, 128, 32, 8, 1, None), (HF, 64, 32, 8, 1, None), (BF, 128, 32, 8, 1, None),
                                                        (HF, 128, 16, 4, 4, 30.0), (HF, 64, 48, 8, 5, None)])
def test_fp16_outputs_lose_their_own_rounding_only(code, io, hd, heads, kvh, sl, softcap):
    """fp16 outputs are off by what rounding the 64-bit result to fp16 costs.  Its errors are
    uniform in a step: their 2-norm over N >= 8192 elements varies by sqrt(0.8 / N) / 2 = 0.5 %
    at most, and what 32-bit sums, a 22-bit probability and the exponential add is 2^-20 of the
    values, a two-hundredth of fp16's 2^-11 / sqrt(3): within 4 %.  Probabilities of 11 bits add a third."""
    A = base._attention()
    gen = torch.Generator().manual_seed(hd + heads)
    cache = base._cache(code, kvh, hd, 32, 16, layers=1)
    lens = [40, 333, 1200, 64, 200, 77]
    state = base._fill(cache, 40, gen)
    ids = torch.stack([torch.randperm(40, generator=gen)[:38] for _ in lens]).to(torch.int32)
    q = torch.randn(len(lens), sl, heads, hd, generator=gen).to(io)
    got = A.kv_attend(q.cuda(), cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=torch.tensor(lens).cuda(),
                      softcap=softcap, out_dtype=HF)
    assert base._status() == 0 and got.dtype == HF
    codes, scales = ko.page_views(state, cache)
    want = torch.stack([ko.attend(q[b], *ko.gather(codes, scales, cache, 0, ids[b], n), [n - sl + 1 + i for i in range(sl)],
                                  hd ** -0.5, softcap) for b, n in enumerate(lens)])
    assert want.numel() >= 8192
    off, least = (got.cpu().double() - want).norm(), (want.half().double() - want).norm()
    assert off <= 1.04 * least, float(off / least)


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io", [BF, HF, F32])
@pytest.mark.parametrize("softcap", [200.0, 300.0, 1e4, 1e6, 1e20])
def test_large_softcaps(code, io, softcap):
    """A cap far above every score leaves the scores as they are."""
    base._attend_case(code, io, 128, 8, 2, 32, 16, [90, 300], softcap=softcap)
    base._attend_case(code, io, 64, 12, 2, 16, 16, [33], sl=3, softcap=softcap)


def _attend_with_scales(code, io, change, lens=(90, 61)):
    """One call over a cache whose V scales [page, layer, head, block] `change` has changed."""
    A = base._attention()
    gen = torch.Generator().manual_seed(21)
    cache = base._cache(code, 2, 128, 32, 16, layers=1)
    state = base._fill(cache, 8, gen)
    sv = state[1].cpu().unflatten(1, cache.scale_page_dims)
    change(sv[..., 1], gen)
    state[1].copy_(sv.flatten(1))
    ids = torch.tensor([[3, 2, 4], [5, 1, 7]], dtype=torch.int32)
    q = torch.randn(2, 1, 8, 128, generator=gen).to(io)
    got = A.kv_attend(q.cuda(), cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=torch.tensor(lens).cuda())
    assert base._status() == 0
    codes, scales = ko.page_views(state, cache)
    for b, n in enumerate(lens):
        k, v = ko.gather(codes, scales, cache, 0, ids[b], n)
        want = ko.attend(q[b], k, v, [n], 128 ** -0.5)
        room = ko.attend_tolerance(q[b], k, v, 128 ** -0.5, 2.0 ** -11 if io == BF else 2.0 ** -21, base.EPS[io], want)
        assert ((got[b].cpu().double() - want).abs() <= room).all(), b


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io", [BF, F32])
def test_values_near_the_end_of_32_bits(code, io):
    """V up to 1.9 * 2^127: 1 / s_v and what the codes are scaled by stay within 32 bits."""
    _attend_with_scales(code, io, lambda s, gen: s.mul_(1.9 * 2.0 ** 127 / ko.QMAX[code] / s.max()))


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io", [BF, F32])
@pytest.mark.parametrize("size", [-60, -30, 0, 30, 48])
def test_blocks_of_zeros_beside_others(code, io, size):
    """Positions whose V is zero keep their weight, however large or small the other values are."""
    def change(s, gen):
        s *= 2.0 ** size
        s[torch.rand(s.shape, generator=gen) < 0.5] = 0.0
    _attend_with_scales(code, io, change)


def test_zeros_and_large_values_in_different_warps():
    """A long sequence: stretches of zeros in some CTAs, values of 2^60 or 2^-60 in others."""
    A = base._attention()
    gen = torch.Generator().manual_seed(22)
    for code, io, size in ((I8, F32, 60), (E4, BF, 60), (E4, F32, -60), (I8, BF, -60)):
        cache = base._cache(code, 1, 64, 32, 16, layers=1)
        state = base._fill(cache, 300, gen)
        sv = state[1].cpu().unflatten(1, cache.scale_page_dims)
        sv[..., 1] *= 2.0 ** size
        sv[:150, ..., 1] = 0.0
        state[1].copy_(sv.flatten(1))
        n = 9000
        for ids in (torch.arange(300), torch.arange(300).flip(0), torch.randperm(300, generator=gen)):
            ids = ids[None].to(torch.int32)
            q = torch.randn(1, 1, 4, 64, generator=gen).to(io)
            got = A.kv_attend(q.cuda(), cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=torch.tensor([n]).cuda())
            assert base._status() == 0
            k, v = ko.gather(*ko.page_views(state, cache), cache, 0, ids[0], n)
            want = ko.attend(q[0], k, v, [n], 64 ** -0.5)
            room = ko.attend_tolerance(q[0], k, v, 64 ** -0.5, 2.0 ** -11 if io == BF else 2.0 ** -21, base.EPS[io], want)
            assert ((got[0].cpu().double() - want).abs() <= room).all(), (code, size)


def test_lengths_written_right_before_the_call():
    """Lengths that the kernel in front of the call writes, in turn long and short ones, give
    what they give on an idle stream: where the joined states are found follows from them."""
    A = base._attention()
    gen = torch.Generator().manual_seed(23)
    cache = base._cache(I8, 2, 64, 16, 16, layers=1)
    state = base._fill(cache, 200, gen)
    bs, per = 5, 190
    ids = torch.stack([torch.randperm(200, generator=gen)[:per] for _ in range(bs)]).to(torch.int32).cuda()
    q = torch.randn(bs, 1, 8, 64, generator=gen).to(BF).cuda()
    attend = lambda lens: A.kv_attend(q, cache, state, block_index=0, seq_block_ids=ids, seq_lens=lens)
    sets = [torch.randint(0, 16 * per, (bs,), generator=gen).to(torch.int32).cuda() for _ in range(12)]
    sets += [torch.full((bs,), n, dtype=torch.int32, device="cuda") for n in (0, 1, 128, 129, 16 * per)]
    want = []
    for x in sets:
        torch.cuda.synchronize()
        want.append(attend(x))
    torch.cuda.synchronize()
    lens = torch.zeros(bs, dtype=torch.int32, device="cuda")
    got = []
    for turn in range(4):
        for i, x in enumerate(sets):
            lens.copy_(x)
            got.append((i, attend(lens)))
            lens.fill_(7)
    assert all(torch.equal(o, want[i]) for i, o in got)
    assert base._status() == 0
