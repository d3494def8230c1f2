"""The 8-bit KV cache on the GPU against its definition in 64 bits: the write (norms,
rotation, quantisation), the read-back and the attention, each alone and together."""
import pytest
import torch

from oracle import kv8_oracle as ko

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half a step of the type's subnormal numbers: fp16 has steps of 2^-24 below 2^-14, which a
# small code times a small scale falls under (2^-9 * 0.01); the others reach below 2^-126
FLOOR = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
I8, E4 = torch.int8, torch.float8_e4m3fn
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _attention():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    from shark_platform_b200 import attention as A

    return A


def _cache(dtype, kvh, hd, stride, block=None, layers=2):
    return _attention().PagedKVCache(transformer_block_count=layers, attn_head_count=kvh, attn_head_dim=hd,
                                     block_seq_stride=stride, dtype=dtype, device="cuda", scale_block=block)


def _freqs(hd):
    return 1.0 / (10000.0 ** (torch.arange(0, hd, 2).float() / hd))


def _fill(cache, pages, gen, std=1.5):
    """Pages that hold quantised normal values everywhere."""
    state = cache.allocate(pages)
    x = torch.randn(pages, *cache.sub_page_dims, generator=gen) * std
    y = x.unflatten(-2, (-1, cache.scale_block))
    s = y.abs().amax(dim=(-1, -2)) / ko.QMAX[cache.dtype]
    c = ko.to_code((y / s[..., None, None]).double(), cache.dtype).float().flatten(-3, -2)
    state[0].copy_(c.to(cache.dtype).view(torch.int8).flatten(1).view(cache.dtype))
    state[1].copy_(s.transpose(-1, -2).reshape(pages, -1))
    return state


def _ids(bs, per, gen):
    return torch.randperm(bs * per + 2, generator=gen)[: bs * per].view(bs, per).to(torch.int32)


def _status():
    from shark_platform_b200 import moe

    return moe.device_status()


# ------------------------------------------------------------------------- write
class Write:
    """One write call and its check against the definition."""

    def __init__(self, cache, heads, io, gen, norm=False, halves=False, std=1.0):
        self.cache, self.heads, self.io, self.gen, self.halves, self.std = cache, heads, io, gen, halves, std
        hd = cache.attn_head_dim
        self.w = [1 + 0.2 * torch.randn(hd, generator=gen) for _ in range(2)] if norm else [None, None]
        self.freqs = _freqs(hd)

    def inputs(self, bs, sl, strided=True):
        kvh, hd = self.cache.attn_head_count, self.cache.attn_head_dim
        qkv = (torch.randn(bs, sl, (self.heads + 2 * kvh) * hd, generator=self.gen) * self.std).to(self.io)
        parts = qkv.split([self.heads * hd, kvh * hd, kvh * hd], dim=-1)
        return qkv, [p.unflatten(-1, (-1, hd)) for p in parts]

    def call(self, state, ids, start, q, k, v, lens=None, layer=1):
        d = lambda t: None if t is None else t.cuda()
        return _attention().norm_rope_kv_write(
            q, k, v, self.cache, state, block_index=layer, seq_block_ids=d(ids), start_positions=d(start),
            new_lens=d(lens), freqs=d(self.freqs), q_norm=d(self.w[0]), k_norm=d(self.w[1]), use_hf=self.halves)

    def rotated(self, start, q, k):
        """64-bit rotated q and k, and how far 32 bits may be from them."""
        sl = q.shape[1]
        pos = start.clamp(min=0)[:, None] + torch.arange(sl)
        out = []
        for x, w in zip((q, k), self.w):
            y = ko.turn(x, pos, self.freqs, w, halves=self.halves)
            # the norm: a sum of hd squares, root and division, two products; the rotation: two
            # products and a sum; cosine and sine to 2^-22 each
            size = x.double().abs().amax(-1, keepdim=True)
            if w is not None:
                size = size * w.abs().max() / x.double().pow(2).mean(-1, keepdim=True).add(1e-5).sqrt()
            out.append((y, size * 16 * 2.0 ** -23))
        return out

    def check(self, before, state, ids, start, q, k, v, got, lens=None, layer=1):
        cache, io = self.cache, self.io
        (q64, dq), (k64, dk) = self.rotated(start, q, k)
        for y, d, g in ((q64, dq, got[0]), (k64, dk, got[1])):
            assert g.shape == y.shape and g.dtype == io and g.is_contiguous()
            off = (g.cpu().double() - y).abs() - d - EPS[io] * (y.abs() + d) - FLOOR[io]
            assert off.max() <= 0, float(off.max())
        bs, sl = q.shape[:2]
        count = [0 if int(start[b]) < 0 else sl if lens is None else min(max(int(lens[b]), 0), sl) for b in range(bs)]
        if not cache.quantized:
            return self._check_plain(before, state, ids, start, k64, dk, v, count, layer)
        c0, s0 = ko.page_views(before, cache)
        c1, s1 = ko.page_views(state, cache)
        stride, blk, qmax = cache.block_seq_stride, cache.scale_block, ko.QMAX[cache.dtype]
        want_c, want_s = c0.clone(), s0.clone()
        for b in range(bs):
            st, n = int(start[b]), count[b]
            if n == 0:
                continue
            for first in range(st // blk * blk, st + n, blk):
                lo, hi = max(first, st), min(first + blk, st + n)
                page, off = int(ids[b, first // stride]), first % stride
                for slot, (x, dx) in enumerate(((k64[b], dk[b]), (v[b].double(), torch.zeros_like(dk[b])))):
                    for h in range(cache.attn_head_count):
                        rows = x[lo - st:hi - st, h]
                        d = dx[lo - st:hi - st, h]
                        amax, da = float(rows.abs().max()), float(d.max())
                        sc = float(s1[page, layer, h, off // blk, slot])
                        old = float(s0[page, layer, h, off // blk, slot]) if lo > first else 0.0
                        if old > 0:
                            grow = round(float(torch.log2(torch.tensor(sc / old)))) if sc > 0 else -1
                            assert grow >= 0 and sc == old * 2.0 ** grow
                            # the power of two is the one the largest value asks for, give or take its error
                            assert ko.growth(amax - da, old, qmax) <= grow <= ko.growth(amax + da, old, qmax)
                            held = c0[page, layer, h, slot, off:off + lo - first]
                            want_c[page, layer, h, slot, off:off + lo - first] = ko.to_code(held * 2.0 ** -grow, cache.dtype)
                        else:
                            assert abs(sc * qmax - amax) <= da + amax * 2.0 ** -22, (sc * qmax, amax)
                        want_s[page, layer, h, off // blk, slot] = sc
                        at = slice(off + lo - first, off + hi - first)
                        code = c1[page, layer, h, slot, at]
                        # nearest code: half a step, the error of the value, of 1 / scale and of the product
                        y = rows / sc if sc > 0 else rows * 0
                        room = ko.half_step(y, cache.dtype) * (1 + 2.0 ** -10) + (d / sc if sc > 0 else 0) + y.abs() * 2.0 ** -22
                        over = (y.abs() - qmax).clamp(min=0)
                        assert ((code - y).abs() - room - over).max() <= 0
                        assert over.max() <= qmax * 2.0 ** -9
                        want_c[page, layer, h, slot, at] = code
        # nothing else has changed
        assert torch.equal(c1.nan_to_num(999.), want_c.nan_to_num(999.))
        assert torch.equal(s1.nan_to_num(-1.), want_s.nan_to_num(-1.))

    def _check_plain(self, before, state, ids, start, k64, dk, v, count, layer):
        cache = self.cache
        view = lambda s: s[0].cpu().unflatten(1, cache.sub_page_dims).clone()
        s0, s1 = view(before), view(state)
        stride = cache.block_seq_stride
        for b, n in enumerate(count):
            for i in range(n):
                p = int(start[b]) + i
                page, off = int(ids[b, p // stride]), p % stride
                y, d = k64[b, i], dk[b, i]
                e = EPS[self.io] + EPS[cache.dtype]
                floor = FLOOR[self.io] + FLOOR[cache.dtype]
                assert ((s1[page, layer, 0, off].double() - y).abs() - d * 2 - e * y.abs() - floor).max() <= 0
                assert torch.equal(s1[page, layer, 1, off], v[b, i].to(cache.dtype))
                s0[page, layer, :, off] = s1[page, layer, :, off]
        assert torch.equal(s0, s1)


def _run_write(w, pages, ids, start, sl, lens=None, fill=True, layer=1, contiguous=False, state=None):
    if state is None:
        state = _fill(w.cache, pages, w.gen) if fill and w.cache.quantized else w.cache.allocate(pages)
    before = [t.clone() for t in state]
    qkv, (q, k, v) = w.inputs(len(start), sl)
    kvh, hd = w.cache.attn_head_count, w.cache.attn_head_dim
    dev = [t.unflatten(-1, (-1, hd)) for t in qkv.cuda().split([w.heads * hd, kvh * hd, kvh * hd], dim=-1)]
    if contiguous:
        dev = [t.contiguous() for t in dev]
    got = w.call(state, ids, start, *dev, lens=lens, layer=layer)
    assert _status() == 0
    assert torch.equal(torch.cat([t.flatten(2) for t in dev], dim=-1).cpu(), qkv)  # inputs as they were
    w.check(before, state, ids, start, q, k, v, got, lens=lens, layer=layer)
    return state


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io,hd,heads,kvh,stride,block,norm,halves", [
    (BF, 128, 8, 2, 32, 16, False, False), (BF, 128, 8, 2, 32, 32, True, True), (HF, 64, 4, 4, 16, 16, True, False),
    (F32, 128, 6, 2, 16, 1, True, True), (F32, 64, 8, 1, 64, 64, False, True), (BF, 64, 12, 1, 20, 4, True, False),
    (HF, 128, 3, 3, 7, 1, False, False), (BF, 128, 4, 1, 8, 2, True, True)])
def test_prompts_and_steps(code, io, hd, heads, kvh, stride, block, norm, halves):
    """Prompts from position 0 and continued ones, ragged with padding, and single tokens."""
    gen = torch.Generator().manual_seed(hd + stride + block)
    cache = _cache(code, kvh, hd, stride, block)
    w = Write(cache, heads, io, gen, norm, halves)
    per = -(-150 // stride)
    ids = _ids(3, per, gen)
    pages = 3 * per + 2
    _run_write(w, pages, ids, torch.tensor([0, 0, 0]), 37, torch.tensor([37, 20, 1]))
    _run_write(w, pages, ids, torch.tensor([5, 16, 33]), 70, torch.tensor([70, 64, 0]), contiguous=True)
    _run_write(w, pages, ids, torch.tensor([0, 17, 149]), 1, layer=0)
    _run_write(w, pages, ids, torch.tensor([1, -1, 64]), 5, fill=False)


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("std", [0.05, 1.0, 40.0, 3000.0])
def test_a_continued_block_grows_by_powers_of_two(code, std):
    """Smaller, equal and larger rows than the block holds already."""
    gen = torch.Generator().manual_seed(11)
    cache = _cache(code, 2, 128, 32, 32)
    w = Write(cache, 4, BF, gen, std=std)
    ids = _ids(4, 3, gen)
    _run_write(w, 14, ids, torch.tensor([1, 31, 40, 70]), 3)
    _run_write(w, 14, ids, torch.tensor([1, 31, 33, 64]), 1)


@pytest.mark.parametrize("code", [I8, E4])
def test_a_block_filled_token_by_token(code):
    """Every row stays within one step of the final scale of what was written: a scale that
    grows by powers of two rounds each code by at most half of each step it passes."""
    A = _attention()
    gen = torch.Generator().manual_seed(3)
    cache = _cache(code, 2, 64, 16, 16)
    state = cache.allocate(3)
    ids = torch.tensor([[1]], dtype=torch.int32).cuda()
    x = torch.randn(16, 2, 64, generator=gen) * torch.exp2(torch.arange(16.)[:, None, None] / 2 - 4)
    for p in range(16):
        t = x[None, p:p + 1].cuda()
        A.norm_rope_kv_write(t, t, t, cache, state, block_index=0, seq_block_ids=ids,
                             start_positions=torch.tensor([p], dtype=torch.int32).cuda(), freqs=_freqs(64).cuda())
    k, v = A.kv_read(cache, state, block_index=0, seq_block_ids=ids, seq_lens=torch.tensor([16]).cuda(), dtype=F32)
    assert _status() == 0
    c, s = ko.page_views(state, cache)
    s = s[1, 0, :, 0]
    for slot, (got, want) in enumerate(((k[0], ko.turn(x, torch.arange(16), _freqs(64))), (v[0], x.double()))):
        sc = s[:, slot][None, :, None]
        # int8: 1/2 + 1/4 + ... of the final step; e4m3: the rounding of the write, then that of subnormal codes
        room = (sc if code == I8 else want.abs() * 2.0 ** -4 + sc * 2.0 ** -9) * (1 + 2.0 ** -10)
        assert ((got.cpu().double() - want).abs() <= room + want.abs() * 2.0 ** -20).all()


@pytest.mark.parametrize("cache_dtype,io", [(BF, BF), (HF, HF), (F32, F32), (F32, BF), (BF, F32), (HF, BF)])
@pytest.mark.parametrize("hd,heads,kvh,stride,norm,halves", [(128, 8, 2, 16, True, False), (64, 6, 3, 20, True, True),
                                                             (128, 4, 4, 32, False, True)])
def test_write_of_a_plain_cache(cache_dtype, io, hd, heads, kvh, stride, norm, halves):
    gen = torch.Generator().manual_seed(hd + stride)
    w = Write(_cache(cache_dtype, kvh, hd, stride), heads, io, gen, norm, halves)
    ids = _ids(3, 5, gen)
    _run_write(w, 17, ids, torch.tensor([0, 5, 19]), 40, torch.tensor([40, 33, 0]))
    _run_write(w, 17, ids, torch.tensor([0, -3, 79]), 1, layer=0)


@pytest.mark.parametrize("order", [False, True])
def test_far_positions(order):
    """Angles of positions where position * freq does not fit 24 bits."""
    gen = torch.Generator().manual_seed(5)
    cache = _cache(I8, 1, 128, 64, 16)
    w = Write(cache, 2, F32, gen, halves=order)
    far = 1_000_003
    ids = torch.zeros(1, far // 64 + 1, dtype=torch.int32)
    ids[0, -1] = 1
    _run_write(w, 3, ids, torch.tensor([far]), 1)


def test_zero_tiny_and_non_finite_rows():
    A = _attention()
    for code in (I8, E4):
        cache = _cache(code, 4, 64, 16, 16)
        state = cache.allocate(2)
        ids = torch.tensor([[1]], dtype=torch.int32).cuda()
        kw = dict(block_index=0, seq_block_ids=ids, freqs=_freqs(64).cuda())
        k = torch.ones(1, 1, 4, 64)
        v = torch.ones(1, 1, 4, 64)
        v[0, 0, 0], v[0, 0, 1], v[0, 0, 2, 5], v[0, 0, 3, 7] = 0.0, 1e-34, float("inf"), float("nan")
        write = lambda p, k, v: A.norm_rope_kv_write(k.cuda(), k.cuda(), v.cuda(), cache, state,
                                                     start_positions=torch.tensor([p]).cuda(), **kw)
        read = lambda n: [t[0].cpu() for t in A.kv_read(cache, state, block_index=0, seq_block_ids=ids,
                                                       seq_lens=torch.tensor([n]).cuda(), dtype=F32)]
        write(0, k, v)
        kk, vv = read(1)
        assert torch.isfinite(kk).all()
        assert (vv[0, 0] == 0).all() and (vv[0, 1] == 0).all() and vv[0, 2].isnan().all() and vv[0, 3].isnan().all()
        write(1, k, torch.full_like(v, 0.25))  # zeros are joined by values; NaN stays until the block is fresh
        vv = read(2)[1]
        assert (vv[0, :2] == 0).all() and (vv[1, :2] == 0.25).all() and vv[:2, 2:].isnan().all()
        write(0, k, torch.full_like(v, 0.5))
        vv = read(1)[1]
        assert (vv[0] == 0.5).all() and (vv[1:] == 0).all()
        assert _status() == 0


def test_padding_rows_do_not_touch_the_cache():
    """NaN in the rows behind new_lens reaches neither codes nor scales."""
    A = _attention()
    cache = _cache(I8, 2, 128, 32, 32)
    gen = torch.Generator().manual_seed(1)
    state, ref = cache.allocate(4), cache.allocate(4)
    x = torch.randn(1, 40, 2, 128, generator=gen).cuda()
    y = x.clone()
    y[:, 35:] = float("nan")
    kw = dict(block_index=1, seq_block_ids=torch.tensor([[2, 1]]).cuda(), freqs=_freqs(128).cuda(),
              start_positions=torch.tensor([0]).cuda())
    A.norm_rope_kv_write(x[:, :35], x[:, :35], x[:, :35], cache, ref, **kw)
    A.norm_rope_kv_write(y, y, y, cache, state, new_lens=torch.tensor([35]).cuda(), **kw)
    assert torch.equal(state[0], ref[0]) and torch.equal(state[1], ref[1])
    assert _status() == 0


@pytest.mark.parametrize("code", [I8, E4, BF])
def test_a_sequence_of_padding_needs_no_pages(code):
    """new_lens 0 in the middle of a scale block: nothing is looked up, written or reported."""
    A = _attention()
    gen = torch.Generator().manual_seed(3)
    cache = _cache(code, 2, 64, 32)
    state = _fill(cache, 3, gen) if cache.quantized else cache.allocate(3)
    before = [t.clone() for t in state]
    x = torch.randn(2, 40, 2, 64, generator=gen).cuda()
    for ids, start in (([[-1, 9], [7, -1]], [5, 37]), ([[0, 1], [1, 2]], [63, 1000])):
        q, k = A.norm_rope_kv_write(x, x, x, cache, state, block_index=0, freqs=_freqs(64).cuda(),
                                    seq_block_ids=torch.tensor(ids).cuda(), start_positions=torch.tensor(start).cuda(),
                                    new_lens=torch.tensor([0, -3]).cuda())
        assert _status() == 0
        assert torch.equal(q, k) and q.isfinite().all()  # rotated all the same
    for t, was in zip(state, before):
        assert torch.equal(t.view(torch.uint8), was.view(torch.uint8))


def test_missing_pages_are_reported_and_skipped():
    from shark_platform_b200 import _cabi as C

    A = _attention()
    gen = torch.Generator().manual_seed(2)
    for code in (I8, BF):
        cache = _cache(code, 2, 64, 16)
        state = cache.allocate(3)
        x = torch.randn(1, 40, 2, 64, generator=gen).cuda()
        kw = dict(block_index=0, freqs=_freqs(64).cuda(), start_positions=torch.tensor([0]).cuda())
        for bad in (7, -1, 2 ** 31 - 1):
            A.norm_rope_kv_write(x, x, x, cache, state, seq_block_ids=torch.tensor([[1, bad, 2]]).cuda(), **kw)
            with pytest.raises(C.B200MoeError, match="status word"):
                _status()
        assert not state[0][0].view(torch.uint8).any() and state[0][1].view(torch.uint8).any()
        # a table too short for the tokens
        A.norm_rope_kv_write(x, x, x, cache, state, seq_block_ids=torch.tensor([[1, 2]]).cuda(), **kw)
        with pytest.raises(C.B200MoeError, match="status word"):
            _status()
        if code == I8:
            ids = torch.tensor([[1, 9, 2]]).cuda()
            lens = torch.tensor([40]).cuda()
            k, v = A.kv_read(cache, state, block_index=0, seq_block_ids=ids, seq_lens=lens, dtype=F32)
            assert (k[0, 16:32] == 0).all() and (k[0, :16] != 0).any() and (k[0, 32:40] != 0).any()
            with pytest.raises(C.B200MoeError, match="status word"):
                _status()
            o = A.kv_attend(x[:, :1], cache, state, block_index=0, seq_block_ids=ids, seq_lens=lens)
            with pytest.raises(C.B200MoeError, match="status word"):
                _status()
            live = [i for i in range(40) if not 16 <= i < 32]
            kk, vv = k[0, live].cpu().double(), v[0, live].cpu().double()
            want = ko.attend(x[0, :1].cpu(), kk, vv, [24], 64 ** -0.5)
            assert ((o[0].cpu().double() - want).abs() <= ko.attend_tolerance(x[0, :1].cpu(), kk, vv, 64 ** -0.5,
                                                                              2.0 ** -22, EPS[F32], want)).all()
    assert _status() == 0


@pytest.mark.parametrize("code", [I8, E4])
def test_stretches_of_missing_pages_are_not_attended(code):
    """Whole steps of positions without a page, in the middle and at the end, and the sequence behind them."""
    from shark_platform_b200 import _cabi as C

    A = _attention()
    gen = torch.Generator().manual_seed(6)
    cache = _cache(code, 2, 128, 16, 16)
    state = _fill(cache, 90, gen)
    ids = torch.stack([torch.arange(40), torch.arange(40, 80)]).to(torch.int32)
    live = ids.clone()
    ids[0, 10:30] = 90
    ids[0, 36:] = -5
    q = torch.randn(2, 1, 8, 128, generator=gen).to(BF)
    o = A.kv_attend(q.cuda(), cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=torch.tensor([637, 640]).cuda())
    with pytest.raises(C.B200MoeError, match="status word"):
        _status()
    codes, scales = ko.page_views(state, cache)
    for b in range(2):
        k, v = ko.gather(codes, scales, cache, 0, live[b], 637 + 3 * b)
        if b == 0:
            keep = [p for p in range(637) if not 160 <= p < 480 and p < 576]
            k, v = k[keep], v[keep]
        want = ko.attend(q[b], k, v, [k.shape[0]], 128 ** -0.5)
        assert ((o[b].cpu().double() - want).abs() <= ko.attend_tolerance(q[b], k, v, 128 ** -0.5, 2.0 ** -11, EPS[BF], want)).all()


def test_a_length_behind_the_page_table_is_reported():
    from shark_platform_b200 import _cabi as C

    A = _attention()
    gen = torch.Generator().manual_seed(6)
    cache = _cache(I8, 1, 64, 16, 16)
    state = _fill(cache, 4, gen)
    ids = torch.tensor([[1, 2]], dtype=torch.int32).cuda()
    q = torch.randn(1, 1, 4, 64, generator=gen).cuda()
    a = A.kv_attend(q, cache, state, block_index=0, seq_block_ids=ids, seq_lens=torch.tensor([32]).cuda())
    assert _status() == 0
    b = A.kv_attend(q, cache, state, block_index=0, seq_block_ids=ids, seq_lens=torch.tensor([33]).cuda())
    with pytest.raises(C.B200MoeError, match="status word"):
        _status()
    assert torch.equal(a, b)
    o = A.kv_attend(q, cache, state, block_index=0, seq_block_ids=ids, seq_lens=torch.tensor([-4]).cuda())
    assert _status() == 0 and not o.any()


@pytest.mark.parametrize("bs", [70, 200])
def test_many_short_sequences(bs):
    """More sequences than one look at the lengths takes, empty ones among them."""
    _attend_case(I8, BF, 64, 8, 4, 16, 16, [(37 * i) % 150 for i in range(bs)])
    _attend_case(E4, F32, 64, 8, 4, 16, 16, [(61 * i) % 300 if i % 7 else 0 for i in range(bs)], sl=2)


# -------------------------------------------------------------------- read-back
@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("dtype", [F32, HF, BF])
@pytest.mark.parametrize("hd,kvh,stride,block,lens", [(128, 2, 32, 16, [1, 77, 0]), (64, 3, 20, 4, [60, 19, 21]),
                                                      (128, 1, 7, 1, [20]), (64, 8, 16, 16, [16, 33])])
def test_read(code, dtype, hd, kvh, stride, block, lens):
    A = _attention()
    gen = torch.Generator().manual_seed(hd + stride)
    cache = _cache(code, kvh, hd, stride, block)
    bs, per = len(lens), -(-max(lens) // stride) + 1
    state = _fill(cache, bs * per + 2, gen)
    ids = _ids(bs, per, gen)
    codes, scales = ko.page_views(state, cache)
    for n in (None, max(lens), 5):
        got = A.kv_read(cache, state, block_index=1, seq_block_ids=ids.cuda(), seq_lens=torch.tensor(lens).cuda(),
                        max_seq_len=n, dtype=dtype)
        assert _status() == 0
        rows = per * stride if n is None else n
        for b, m in enumerate(lens):
            m = min(m, rows)
            want = ko.gather(codes, scales, cache, 1, ids[b], m)
            for slot, g in enumerate(got):
                assert g.shape == (bs, rows, kvh, hd) and g.dtype == dtype
                # one product of exact numbers, rounded to 32 bits and to the type
                off = (g[b, :m].cpu().double() - want[slot]).abs()
                over = off - want[slot].abs() * (EPS[dtype] * (1 + 2.0 ** -8) + 2.0 ** -24) - FLOOR[dtype]
                assert m == 0 or over.max() <= 0
                assert (g[b, m:] == 0).all()


# -------------------------------------------------------------------- attention
def _attend_case(code, io, hd, heads, kvh, stride, block, lens, sl=1, softcap=None, scale=None, qstd=1.0, kstd=1.5,
                 out=None, seed=0, poison=True):
    A = _attention()
    gen = torch.Generator().manual_seed(hd + stride + heads + seed)
    cache = _cache(code, kvh, hd, stride, block)
    bs, per = len(lens), -(-max(max(lens), 1) // stride) + 1
    ids = _ids(bs, per, gen)
    state = _fill(cache, bs * per + 2, gen, std=kstd)
    codes, scales = ko.page_views(state, cache)
    if poison:  # what no row attends: NaN codes behind the lengths, NaN scales of blocks and pages that are not live
        cv = state[0].view(torch.int8).unflatten(1, cache.sub_page_dims)
        sv = state[1].unflatten(1, cache.scale_page_dims)
        for b, n in enumerate(lens):
            for p in range(n, per * stride):
                cv[int(ids[b, p // stride]), :, :, :, p % stride] = 127  # e4m3: NaN
                if p % block == 0:
                    sv[int(ids[b, p // stride]), :, :, (p % stride) // block] = float("nan")
    q = (torch.randn(bs, sl, heads, hd, generator=gen) * qstd).to(io)
    got = A.kv_attend(q.cuda(), cache, state, block_index=1, seq_block_ids=ids.cuda(), seq_lens=torch.tensor(lens).cuda(),
                      softcap=softcap, scale=scale, out_dtype=out)
    assert _status() == 0
    out = io if out is None else out
    assert got.shape == q.shape and got.dtype == out
    scale = hd ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        k, v = ko.gather(codes, scales, cache, 1, ids[b], n)
        seen = [n - sl + 1 + i for i in range(sl)]
        want = ko.attend(q[b], k, v, seen, scale, softcap)
        # 16-bit activations: probabilities in fp16; 32-bit ones: in two fp16 parts
        room = ko.attend_tolerance(q[b], k, v, scale, 2.0 ** -11 if io != F32 else 2.0 ** -21, EPS[out], want) + FLOOR[out]
        off = (got[b].cpu().double() - want).abs()
        assert bool((off <= room).all()), (b, n, float((off / room).max()))
        for i, m in enumerate(seen):
            if m <= 0:
                assert (got[b, i] == 0).all()


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io", [BF, HF, F32])
@pytest.mark.parametrize("hd,heads,kvh,stride,block,lens", [
    (128, 8, 2, 32, 16, [1, 0, 15, 16, 17, 31, 32, 33]), (64, 4, 4, 16, 16, [63, 64, 65, 127, 128, 129, 300]),
    (128, 8, 1, 64, 64, [1000, 513]), (64, 16, 4, 20, 4, [201, 40, 19]), (128, 3, 3, 7, 1, [50, 7, 8]),
    (64, 32, 1, 16, 1, [100]), (128, 24, 2, 32, 8, [70, 3])])
def test_attend_one_token(code, io, hd, heads, kvh, stride, block, lens):
    _attend_case(code, io, hd, heads, kvh, stride, block, lens)


@pytest.mark.parametrize("code,io", [(I8, BF), (E4, F32), (E4, HF)])
@pytest.mark.parametrize("sl", [2, 3, 5, 8, 16])
@pytest.mark.parametrize("hd,heads,kvh,stride,block", [(128, 8, 2, 32, 16), (64, 6, 1, 20, 4), (128, 2, 2, 16, 1)])
def test_attend_several_tokens(code, io, sl, hd, heads, kvh, stride, block):
    _attend_case(code, io, hd, heads, kvh, stride, block, [sl, 200, sl + 1, 64 + sl, sl - 1, 1, 0], sl=sl)


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io", [BF, F32])
def test_attend_softcap_scale_and_output_type(code, io):
    _attend_case(code, io, 128, 8, 2, 32, 16, [90, 300], softcap=30.0)
    _attend_case(code, io, 128, 8, 2, 32, 16, [90, 300], sl=2, softcap=0.5, scale=0.3)
    _attend_case(code, io, 64, 8, 8, 16, 16, [33], scale=-0.2, out=HF)
    _attend_case(code, io, 128, 8, 2, 32, 16, [90, 300], scale=0.0)


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("qstd,kstd", [(1e-4, 1.0), (2000.0, 1e-3), (1.0, 1e-6), (1e-3, 1e4), (30.0, 1.0)])
def test_attend_ranges(code, qstd, kstd):
    """Queries and scales far from one; scores that make the softmax one position."""
    _attend_case(code, BF, 128, 8, 2, 32, 16, [150, 16], qstd=qstd, kstd=kstd)
    _attend_case(code, F32, 64, 4, 1, 16, 4, [150, 16], qstd=qstd, kstd=kstd)


@pytest.mark.parametrize("io,heads,kvh,hd,block", [(BF, 8, 1, 128, 16), (F32, 8, 2, 64, 1), (HF, 8, 8, 128, 32)])
def test_attend_long(io, heads, kvh, hd, block):
    _attend_case(I8, io, hd, heads, kvh, 32, block, [5003], poison=False)
    _attend_case(E4, io, hd, heads, kvh, 32, block, [2048, 2049, 31], poison=False)


@pytest.mark.parametrize("code", [I8, E4])
def test_scales_that_differ_by_much(code):
    """Blocks of one sequence whose K and V differ by up to 2^40 in size, and empty ones."""
    A = _attention()
    gen = torch.Generator().manual_seed(9)
    cache = _cache(code, 2, 128, 32, 16)
    state = _fill(cache, 5, gen)
    sv = state[1].unflatten(1, cache.scale_page_dims)
    size = torch.exp2(torch.randint(-20, 21, sv.shape, generator=gen).float())
    size[..., 0] = 1.0                       # K as it is: all positions count
    size[2, :, 0, 0, 1] = 0.0                # a block of zeros
    sv *= size.cuda()
    ids = torch.tensor([[3, 2, 4]], dtype=torch.int32)
    codes, scales = ko.page_views(state, cache)
    for io in (BF, F32):
        q = torch.randn(1, 1, 8, 128, generator=gen).to(io)
        got = A.kv_attend(q.cuda(), cache, state, block_index=1, seq_block_ids=ids.cuda(), seq_lens=torch.tensor([90]).cuda())
        k, v = ko.gather(codes, scales, cache, 1, ids[0], 90)
        want = ko.attend(q[0], k, v, [90], 128 ** -0.5)
        off = (got[0].cpu().double() - want).abs()
        for h in range(8):  # per kv head: the largest V of its own
            room = ko.attend_tolerance(q[0, :, h:h + 1], k[:, h // 4:h // 4 + 1], v[:, h // 4:h // 4 + 1], 128 ** -0.5,
                                       2.0 ** -11 if io != F32 else 2.0 ** -21, EPS[io], want[:, h:h + 1])
            assert (off[:, h:h + 1] <= room).all()
    assert _status() == 0


def test_a_nan_block_shows_where_it_is_attended_only():
    A = _attention()
    gen = torch.Generator().manual_seed(4)
    cache = _cache(I8, 2, 64, 16, 16)
    state = _fill(cache, 6, gen)
    state[1].unflatten(1, cache.scale_page_dims)[2, 1, 0, 0, :] = float("nan")  # page 2, kv head 0
    ids = torch.tensor([[1, 2], [3, 4]], dtype=torch.int32).cuda()
    q = torch.randn(2, 1, 4, 64, generator=gen).cuda()
    o = A.kv_attend(q, cache, state, block_index=1, seq_block_ids=ids, seq_lens=torch.tensor([20, 20]).cuda())
    assert o[0, 0, :2].isnan().all() and torch.isfinite(o[0, 0, 2:]).all() and torch.isfinite(o[1]).all()
    o = A.kv_attend(q, cache, state, block_index=1, seq_block_ids=ids, seq_lens=torch.tensor([16, 20]).cuda())
    assert torch.isfinite(o).all()
    assert _status() == 0


# ------------------------------------------------------------------- all together
@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("io", [BF, F32])
def test_a_serving_run(code, io):
    """Prompts, single tokens and drafted tokens: every step's attention against the values
    that the cache then holds, and those against what was written."""
    A = _attention()
    gen = torch.Generator().manual_seed(7)
    hd, heads, kvh, stride = 128, 8, 2, 32
    cache = _cache(code, kvh, hd, stride, 16, layers=1)
    w = Write(cache, heads, io, gen, norm=True, halves=True)
    ids = _ids(2, 4, gen)
    state = cache.allocate(10)
    done = torch.tensor([0, 0])
    for sl, lens in ((45, [45, 30]), (1, None), (1, None), (4, None), (1, None)):
        qkv, (q, k, v) = w.inputs(2, sl)
        dev = [t.unflatten(-1, (-1, hd)) for t in qkv.cuda().split([heads * hd, kvh * hd, kvh * hd], dim=-1)]
        before = [t.clone() for t in state]
        news = None if lens is None else torch.tensor(lens)
        got = w.call(state, ids, done, *dev, lens=news, layer=0)
        w.check(before, state, ids, done, q, k, v, got, lens=news, layer=0)
        done = done + (sl if lens is None else news)
        kk, vv = A.kv_read(cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=done.cuda(), dtype=F32)
        if sl <= 16:
            o = A.kv_attend(got[0], cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=done.cuda())
            for b in range(2):
                n = int(done[b])
                kb, vb = kk[b, :n].cpu().double(), vv[b, :n].cpu().double()
                want = ko.attend(got[0][b].cpu(), kb, vb, [n - sl + 1 + i for i in range(sl)], hd ** -0.5)
                room = ko.attend_tolerance(got[0][b].cpu(), kb, vb, hd ** -0.5, 2.0 ** -11 if io != F32 else 2.0 ** -21,
                                           EPS[io], want)
                assert ((o[b].cpu().double() - want).abs() <= room).all()
    assert _status() == 0


def _step(A, cache, state, ids, start, q, k, v, freqs):
    qr, _ = A.norm_rope_kv_write(q, k, v, cache, state, block_index=0, seq_block_ids=ids, start_positions=start, freqs=freqs)
    return A.kv_attend(qr, cache, state, block_index=0, seq_block_ids=ids, seq_lens=start + q.shape[1])


def test_captured_steps_and_other_streams():
    """Two graphs of a decode step, replayed in turn with new tokens, and the same steps on
    another stream, give what plain calls give, bit for bit."""
    A = _attention()
    gen = torch.Generator().manual_seed(8)
    cache = _cache(E4, 2, 128, 32, 16, layers=1)
    bs, heads, hd = 3, 8, 128
    ids = _ids(bs, 3, gen).cuda()
    freqs = _freqs(hd).cuda()
    steps = [[(torch.randn(bs, 1, n, hd, generator=gen)).to(BF).cuda() for n in (heads, 2, 2)] for _ in range(6)]
    starts = [torch.tensor([10 + i, 40 + i, 63 + i], dtype=torch.int32).cuda() for i in range(6)]
    begin = _fill(cache, 12, gen)
    fresh = lambda: [t.clone() for t in begin]

    ref_state = fresh()
    ref = [_step(A, cache, ref_state, ids, p, *x, freqs) for p, x in zip(starts, steps)]

    side, state = torch.cuda.Stream(), fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_step(A, cache, state, ids, p, *x, freqs) for p, x in zip(starts, steps)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(ref_state, state))

    state = fresh()
    inputs = [[t.clone() for t in steps[0]] for _ in range(2)]
    pos = [starts[0].clone() for _ in range(2)]
    graphs, outs = [], []
    for g in range(2):
        warm = fresh()
        _step(A, cache, warm, ids, pos[g], *inputs[g], freqs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(A, cache, state, ids, pos[g], *inputs[g], freqs))
        graphs.append(graph)
    for a, b in zip(state, begin):
        a.copy_(b)
    for i, (p, x) in enumerate(zip(starts, steps)):
        g = i % 2
        pos[g].copy_(p)
        for t, u in zip(inputs[g], x):
            t.copy_(u)
        graphs[g].replay()
        assert torch.equal(outs[g], ref[i]), i
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(ref_state, state))
    assert _status() == 0


def test_a_slab_beyond_four_gigabytes():
    """Pages whose codes lie behind 2^32 bytes, written, read and attended."""
    A = _attention()
    gen = torch.Generator().manual_seed(12)
    cache = _cache(I8, 8, 128, 64, 16)
    pages = (1 << 32) // cache.page_slab_flat_dim + 40
    state = cache.allocate(pages)
    w = Write(cache, 8, BF, gen)
    ids = torch.tensor([[pages - 1, pages - 30], [pages - 2, 0]], dtype=torch.int32)
    _, (q, k, v) = w.inputs(2, 90)
    zero = torch.zeros(2, dtype=torch.int32)
    got = w.call(state, ids, zero, q.cuda(), k.cuda(), v.cuda())
    low = cache.allocate(4)
    near = torch.tensor([[3, 2], [1, 0]], dtype=torch.int32)
    w.call(low, near, zero, q.cuda(), k.cuda(), v.cuda())
    lens = torch.tensor([90, 77]).cuda()
    for f in (lambda st, i: A.kv_read(cache, st, block_index=1, seq_block_ids=i.cuda(), seq_lens=lens),
              lambda st, i: [A.kv_attend(got[0][:, -1:], cache, st, block_index=1, seq_block_ids=i.cuda(), seq_lens=lens)]):
        assert all(torch.equal(a, b) for a, b in zip(f(state, ids), f(low, near)))
    assert _status() == 0


def test_calls_on_two_streams_at_once():
    """Long and short calls that overlap give what each gives alone."""
    A = _attention()
    gen = torch.Generator().manual_seed(13)
    cache = _cache(E4, 4, 128, 32, 16, layers=1)
    per = 130
    state = _fill(cache, 4 * per + 2, gen)
    ids = _ids(4, per, gen).cuda()
    jobs = []
    for i, (n, sl) in enumerate(((4100, 1), (300, 4), (33, 1), (2000, 8))):
        q = torch.randn(4, sl, 16, 128, generator=gen).to(BF).cuda()
        lens = torch.tensor([n, n // 2 + 8, n, 9]).cuda()
        jobs.append(lambda q=q, lens=lens: A.kv_attend(q, cache, state, block_index=0, seq_block_ids=ids, seq_lens=lens))
    alone = [j() for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(6):
        for i, j in enumerate(jobs):
            with torch.cuda.stream(streams[(i + turn) % 2]):
                got.append((i, j()))
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone[i]) for i, o in got)
    assert _status() == 0


@pytest.mark.parametrize("sl", [1, 4])
def test_new_tokens_behind_the_page_table(sl):
    """Drafted tokens that would not fit are reported; the tokens before them see what they should."""
    from shark_platform_b200 import _cabi as C

    A = _attention()
    gen = torch.Generator().manual_seed(14)
    cache = _cache(I8, 2, 64, 16, 16, layers=1)
    state = _fill(cache, 4, gen)
    ids = torch.tensor([[1, 3]], dtype=torch.int32).cuda()
    q = torch.randn(1, sl, 4, 64, generator=gen).cuda()
    o = A.kv_attend(q, cache, state, block_index=0, seq_block_ids=ids, seq_lens=torch.tensor([32 + sl - 1]).cuda())
    if sl > 1:
        with pytest.raises(C.B200MoeError, match="status word"):
            _status()
    first = A.kv_attend(q[:, :1], cache, state, block_index=0, seq_block_ids=ids, seq_lens=torch.tensor([32]).cuda())
    assert _status() == 0
    k, v = (t[0].cpu().double() for t in A.kv_read(cache, state, block_index=0, seq_block_ids=ids,
                                                  seq_lens=torch.tensor([32]).cuda(), dtype=F32))
    want = ko.attend(q[0, :1].cpu(), k, v, [32], 64 ** -0.5)
    room = ko.attend_tolerance(q[0, :1].cpu(), k, v, 64 ** -0.5, 2.0 ** -21, EPS[F32], want)
    for got in (o[0, :1], first[0]):
        assert ((got.cpu().double() - want).abs() <= room).all()


def test_orders_and_alignments_of_the_inputs():
    """Transposed, expanded, offset and sliced tensors, 64-bit and sliced index tensors, give
    what contiguous ones give."""
    A = _attention()
    gen = torch.Generator().manual_seed(15)
    cache = _cache(E4, 2, 64, 16, 8, layers=1)
    ids = torch.tensor([[1, 4, 2], [5, 0, 3]], dtype=torch.int32).cuda()
    q, k, v = (torch.randn(2, 20, h, 64, generator=gen).to(BF).cuda() for h in (8, 2, 2))
    k = k[:1].expand(2, -1, -1, -1).contiguous()
    start = torch.tensor([3, 0], dtype=torch.int32).cuda()
    lens = torch.tensor([23, 20], dtype=torch.int32).cuda()

    def off(t):  # starts two bytes behind a 16-byte boundary
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
        return flat.copy_(t.reshape(-1)).view_as(t)

    variants = {
        "transposed": (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),) * 3,
        "offset": (off, off, off),
        "wide rows": (lambda t: torch.cat([t, t], dim=-1)[..., :64],) * 3,
        "expanded": (lambda t: t, lambda t: t[:1].expand(2, -1, -1, -1), lambda t: t),
        "padded rows": (lambda t: torch.cat([t.flatten(2), t.flatten(2)[..., :3]], dim=-1)[..., :-3].unflatten(-1, (-1, 64)),) * 3,
    }

    def go(q, k, v, ids, start, lens):
        state = cache.allocate(6)
        a, b = A.norm_rope_kv_write(q, k, v, cache, state, block_index=0, seq_block_ids=ids, start_positions=start,
                                    freqs=_freqs(64).cuda())
        o = A.kv_attend(q[:, :5], cache, state, block_index=0, seq_block_ids=ids, seq_lens=lens)
        return [a, b, o, state[0].view(torch.int8), state[1], *A.kv_read(cache, state, block_index=0, seq_block_ids=ids, seq_lens=lens)]

    want = go(q, k, v, ids, start, lens)
    for name, fs in variants.items():
        for x, y in zip(want, go(*(f(t) for f, t in zip(fs, (q, k, v))), ids, start, lens)):
            assert torch.equal(x, y), name
    wide = torch.cat([ids, ids], dim=1).long()[:, :3]
    for x, y in zip(want, go(q, k, v, wide, start.long(), torch.stack([lens, lens], dim=1)[:, 0])):
        assert torch.equal(x, y)
    assert _status() == 0


def test_rows_of_no_tokens():
    A = _attention()
    cache = _cache(I8, 2, 64, 16, layers=1)
    state = cache.allocate(2)
    e = lambda *s: torch.empty(*s, dtype=BF, device="cuda")
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    for bs, sl in ((0, 4), (2, 0)):
        a, b = A.norm_rope_kv_write(e(bs, sl, 4, 64), e(bs, sl, 2, 64), e(bs, sl, 2, 64), cache, state, block_index=0,
                                    seq_block_ids=i(bs, 1), start_positions=i(bs), freqs=_freqs(64).cuda())
        assert a.shape == (bs, sl, 4, 64) and b.shape == (bs, sl, 2, 64)
    assert A.kv_attend(e(0, 1, 4, 64), cache, state, block_index=0, seq_block_ids=i(0, 1), seq_lens=i(0)).shape == (0, 1, 4, 64)
    k, v = A.kv_read(cache, state, block_index=0, seq_block_ids=i(2, 1), seq_lens=i(2), max_seq_len=0)
    assert k.shape == v.shape == (2, 0, 2, 64)
    k, v = A.kv_read(cache, state, block_index=0, seq_block_ids=i(2, 1), seq_lens=i(2))
    assert not k.any() and not v.any()
    assert _status() == 0
