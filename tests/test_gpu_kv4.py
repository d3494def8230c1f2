"""The 4-bit KV cache on the GPU against its definition in 64 bits: the write (norms, rotation,
quantisation), the read-back and the attention, each alone and together with the prompt
attention."""
import math

import pytest
import torch

from oracle import kv4_oracle as k4, kv8_oracle as ko, prompt_oracle as po

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half a step of the type's subnormal numbers
FLOOR = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _attention():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    from shark_platform_b200 import attention as A

    return A


def _status():
    from shark_platform_b200 import moe

    return moe.device_status()


def _cache(kvh, hd, stride, layers=2):
    return _attention().PagedKVCache(transformer_block_count=layers, attn_head_count=kvh, attn_head_dim=hd,
                                     block_seq_stride=stride, dtype=torch.uint8, device="cuda")


def _ids(bs, per, gen):
    return torch.randperm(bs * per + 2, generator=gen)[: bs * per].view(bs, per).to(torch.int32)


def _freqs(hd):
    return 1.0 / (10000.0 ** (torch.arange(0, hd, 2).float() / hd))


# ------------------------------------------------------------------------- write
def _check_write(cache, before, state, ids, start, q, k, v, got, norms, halves, lens=None, layer=1):
    io, hd, stride = q.dtype, q.shape[-1], cache.block_seq_stride
    bs, sl = q.shape[:2]
    pos = start.clamp(min=0)[:, None] + torch.arange(sl)
    rotated = []
    for x, w, g in ((q, norms[0], got[0]), (k, norms[1], got[1])):
        y = ko.turn(x, pos, _freqs(hd), w, halves=halves)
        # as for the 8-bit cache: a sum of hd squares, root and division, two products; two products
        # and a sum; cosine and sine
        size = x.double().abs().amax(-1, keepdim=True)
        if w is not None:
            size = size * w.abs().max() / x.double().pow(2).mean(-1, keepdim=True).add(1e-5).sqrt()
        d = size * 16 * 2.0 ** -23
        off = (g.cpu().double() - y).abs() - d - EPS[io] * (y.abs() + d) - FLOOR[io]
        assert g.shape == y.shape and g.dtype == io and g.is_contiguous() and off.max() <= 0, float(off.max())
        rotated.append((y, d))
    c0, h0 = k4.page_views(before, cache)
    c1, h1 = k4.page_views(state, cache)
    for b in range(bs):
        n = 0 if int(start[b]) < 0 else sl if lens is None else min(max(int(lens[b]), 0), sl)
        if n == 0:
            continue
        p = pos[b, :n]
        at = (ids[b].long()[p // stride], layer)
        for slot, (x, d) in enumerate(((rotated[1][0][b, :n], rotated[1][1][b, :n]),
                                       (v[b, :n].double(), torch.zeros_like(rotated[1][1][b, :n])))):
            held, code = h1[at[0], layer, :, slot, p % stride], c1[at[0], layer, :, slot, p % stride]
            y = k4.groups(x)
            lo, hi = y.amin(-1), y.amax(-1)
            # the scale: twice the values' error, a difference and a quotient in 32 bits, the rounding to fp16
            want = (hi - lo) / 15
            assert ((held[..., 0] - want).abs() - 2 * d / 15 - (want + d) * (2.0 ** -22 + 2.0 ** -11) - 2.0 ** -25).max() <= 0
            assert ((held[..., 1] - lo).abs() - d - lo.abs() * 2.0 ** -11 - 2.0 ** -25).max() <= 0
            # codes: half a step, the value's error, and the quotient's in 32 bits
            z = k4.quotients(x, held)
            s = held[..., 0].repeat_interleave(k4.GROUP, -1)
            step = torch.where(s > 0, d / s.clamp(min=1e-30), torch.zeros_like(s))
            over = (z - 15).clamp(min=0) + (-z).clamp(min=0)
            assert ((code - z).abs() - 0.5 - step - over - 2.0 ** -19).max() <= 0
            # a scale rounded down leaves the largest value 2^-11 of 15 steps above the last code, a
            # scale among fp16's subnormal numbers more; so does an offset rounded by 2^-11 of itself:
            # hi - offset = 15 (hi - lo) / 15 + lo - offset
            least = lo.abs().repeat_interleave(k4.GROUP, -1)
            assert ((over - step) * s - 15 * (s * 2.0 ** -11 + 2.0 ** -25) * 1.001 - least * 2.0 ** -11 - 2.0 ** -23).max() <= 0
            c0[at[0], layer, :, slot, p % stride], h0[at[0], layer, :, slot, p % stride] = code, held
    # nothing else has changed
    assert torch.equal(c0, c1) and torch.equal(h0.nan_to_num(7e5), h1.nan_to_num(7e5))


def _write(cache, state, ids, start, q, k, v, norms=(None, None), halves=False, lens=None, layer=1):
    c = lambda t: None if t is None else t.cuda()
    return _attention().norm_rope_kv_write(q, k, v, cache, state, block_index=layer, seq_block_ids=c(ids),
                                           start_positions=c(start), new_lens=c(lens), freqs=c(_freqs(q.shape[-1])),
                                           q_norm=c(norms[0]), k_norm=c(norms[1]), use_hf=halves)


@pytest.mark.parametrize("io", [BF, HF, F32])
@pytest.mark.parametrize("heads,kvh,hd,stride", [(8, 2, 128, 32), (4, 4, 64, 16), (3, 1, 128, 7), (12, 3, 64, 5), (40, 8, 128, 32)])
@pytest.mark.parametrize("norm,halves", [(False, False), (True, True)])
def test_write(io, heads, kvh, hd, stride, norm, halves):
    gen = torch.Generator().manual_seed(heads * stride + hd)
    cache = _cache(kvh, hd, stride)
    norms = [1 + 0.2 * torch.randn(hd, generator=gen) for _ in range(2)] if norm else [None, None]
    for bs, sl, lens in ((1, 1, None), (3, 1, None), (2, 37, [37, 20]), (3, 5, [0, 5, 9]), (1, 130, None)):
        start = torch.randint(0, 60, (bs,), generator=gen)
        if bs == 3:
            start[1] = -1 if sl == 1 else start[1]
        per = (60 + sl) // stride + 1
        ids = _ids(bs, per, gen)
        state = k4.fill(cache, bs * per + 2, gen)
        before = [t.clone() for t in state]
        qkv = torch.randn(bs, sl, (heads + 2 * kvh) * hd, generator=gen).to(io).cuda()
        q, k, v = (p.unflatten(-1, (-1, hd)) for p in qkv.split([heads * hd, kvh * hd, kvh * hd], dim=-1))
        was = qkv.clone()
        lens = None if lens is None else torch.tensor(lens)
        got = _write(cache, state, ids, start, q, k, v, norms, halves, lens)
        assert torch.equal(qkv, was)
        _check_write(cache, before, state, ids, start, q.cpu(), k.cpu(), v.cpu(), got, norms, halves, lens)
    assert _status() == 0


def test_write_ties_and_flat_rows():
    """Quotients halfway between codes go to the even one; a row of one value has scale 0 and reads as it."""
    cache = _cache(1, 64, 4, layers=1)
    state = cache.allocate(1)
    v = torch.zeros(1, 3, 1, 64)
    v[0, 0, 0, :32] = torch.arange(32) * 0.5 % 15.5      # 0, .5, 1 .. 15: scale 1
    v[0, 0, 0, 32:] = 0.375                              # flat
    v[0, 1, 0] = torch.tensor([-2.0, 13.0]).repeat(32)   # scale 1, offset -2
    v[0, 2, 0] = torch.arange(64) * 2.0 ** -24           # fp16's smallest steps
    x = v.to(F32).cuda()
    _write(cache, state, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), x, x, x, layer=0)
    c, h = k4.page_views(state, cache)
    c, h = c[0, 0, 0, 1], h[0, 0, 0, 1]
    assert h[0, 0].tolist() == [1.0, 0.0] and h[0, 1].tolist() == [0.0, 0.375] and h[1, 0].tolist() == [1.0, -2.0]
    assert torch.equal(c[0, :32], torch.round(v[0, 0, 0, :32].double())) and not c[0, 32:].any()
    assert torch.equal(c[1], torch.tensor([0.0, 15.0]).repeat(32).double())
    k, v2 = _attention().kv_read(cache, state, block_index=0, seq_block_ids=torch.zeros(1, 1, dtype=torch.int32).cuda(),
                                 seq_lens=torch.tensor([3]).cuda(), dtype=F32)
    assert torch.equal(v2[0, 0, 0, 32:].cpu(), v[0, 0, 0, 32:])
    assert (v2[0, 2, 0].cpu() - v[0, 2, 0]).abs().max() <= 2.0 ** -23


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, -7e4, 2e6])
@pytest.mark.parametrize("halves", [False, True])
def test_bad_values_fill_their_group(bad, halves):
    """Infinities, NaN and scales or offsets that fp16 does not hold: their 32 values read as NaN, no others, until written again."""
    A = _attention()
    cache = _cache(2, 128, 16, layers=1)
    state = cache.allocate(3)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(1, 20, 2, 128, generator=g) for _ in range(2))
    ids, zero = torch.tensor([[2, 0]], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    v[0, 5, 1, 70] = bad
    k[0, 0, 0, 3] = bad  # position 0: not rotated
    read = lambda: [t[0].cpu() for t in A.kv_read(cache, state, block_index=0, seq_block_ids=ids.cuda(),
                                                   seq_lens=torch.tensor([20]).cuda(), max_seq_len=20, dtype=F32)]
    _write(cache, state, ids, zero, k.cuda(), k.cuda(), v.cuda(), halves=halves, layer=0)
    kk, vv = read()
    lost = torch.zeros(20, 2, 128, dtype=torch.bool)
    lost[5, 1, 64:96] = True
    assert torch.equal(torch.isnan(vv), lost)
    lost_k = torch.zeros_like(lost)
    lost_k[0, 0, :32] = True
    if math.isfinite(bad):
        assert torch.equal(torch.isnan(kk), lost_k)
    else:  # infinity times the sine of 0 is NaN: its partner of the rotation too
        lost_k[0, 0, 64:96] = halves
        assert torch.equal(torch.isnan(kk), lost_k)
    v[0, 5, 1, 70], k[0, 0, 0, 3] = 0, 0
    _write(cache, state, ids, zero, k.cuda(), k.cuda(), v.cuda(), halves=halves, layer=0)
    assert all(torch.isfinite(t).all() for t in read())


def test_missing_pages():
    """A missing page: neither written nor read nor attended; the status word says so."""
    from shark_platform_b200 import _cabi as C

    A = _attention()
    gen = torch.Generator().manual_seed(2)
    cache = _cache(2, 64, 8)
    state = k4.fill(cache, 6, gen)
    before = [t.clone() for t in state]
    k = torch.randn(1, 24, 2, 64, generator=gen).cuda()
    ids = torch.tensor([[3, 77, 1]], dtype=torch.int32)
    _write(cache, state, ids, torch.zeros(1, dtype=torch.int32), k, k, k)
    with pytest.raises(C.B200MoeError, match="status word"):
        _status()
    changed = (state[0] != before[0]).any(1).cpu()
    assert changed.tolist() == [False, True, False, True, False, False]
    # tokens behind the page table are not written either
    _write(cache, state, ids[:, :1], torch.tensor([4], dtype=torch.int32), k[:, :6], k[:, :6], k[:, :6])
    with pytest.raises(C.B200MoeError, match="status word"):
        _status()
    kk, vv = A.kv_read(cache, state, block_index=1, seq_block_ids=ids.cuda(), seq_lens=torch.tensor([24]).cuda(), dtype=F32)
    assert not kk[0, 8:16].any() and not vv[0, 8:16].any() and kk[0, 16:].any()
    with pytest.raises(C.B200MoeError, match="status word"):
        _status()
    q = torch.randn(1, 1, 4, 64, generator=gen)
    got = A.kv_attend(q.cuda(), cache, state, block_index=1, seq_block_ids=ids.cuda(), seq_lens=torch.tensor([24]).cuda())
    with pytest.raises(C.B200MoeError, match="status word"):
        _status()
    keep = [p for p in range(24) if p // 8 != 1]
    want = ko.attend(q[0], kk[0].cpu().double()[keep], vv[0].cpu().double()[keep], [16], 1 / 8)
    assert (got[0].cpu().double() - want).abs().max() < 1e-5
    assert _status() == 0


# -------------------------------------------------------------------------- read
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("hd,stride", [(128, 32), (64, 16), (128, 7), (64, 5)])
def test_read(dtype, hd, stride):
    gen = torch.Generator().manual_seed(stride)
    cache = _cache(3, hd, stride)
    ids = _ids(3, 9, gen)
    state = k4.fill(cache, 29, gen)
    lens = torch.tensor([9 * stride, 0, 4 * stride + 1])
    for rows in (None, 2 * stride + 3, 1):
        n = 9 * stride if rows is None else rows
        k, v = _attention().kv_read(cache, state, block_index=1, seq_block_ids=ids.cuda(), seq_lens=lens.cuda(),
                                    max_seq_len=rows, dtype=dtype)
        codes, held = k4.page_views(state, cache)
        for b in range(3):
            want = k4.gather(codes, held, cache, 1, ids[b], n)
            want[:, int(lens[b]):] = 0
            for got, w in ((k[b], want[0]), (v[b], want[1])):
                # the value is exact in 32 bits but for one rounding of the sum, then the type's
                off = (got.cpu().double() - w).abs() - w.abs() * (EPS[dtype] + 2.0 ** -24) * (1 + 2.0 ** -20) - FLOOR[dtype]
                assert got.shape == w.shape and got.dtype == dtype and off.max() <= 0
    assert _status() == 0


# ------------------------------------------------------------------------ attend
def _attend_check(cache, state, ids, lens, q, layer=1, softcap=None, scale=None, out_dtype=None):
    got = _attention().kv_attend(q.cuda(), cache, state, block_index=layer, seq_block_ids=ids.cuda(), seq_lens=lens.cuda(),
                                 scale=scale, softcap=softcap, out_dtype=out_dtype)
    out_dtype = out_dtype or q.dtype
    assert got.shape == q.shape and got.dtype == out_dtype and got.is_contiguous()
    codes, held = k4.page_views(state, cache)
    scale = scale or 1 / math.sqrt(q.shape[-1])
    # bf16 outputs: P to 2^-12 and its product with a scale again; else (and for 32-bit q) 2^-22
    p_eps = 2.0 ** -11 if out_dtype == BF and q.dtype != F32 else 2.0 ** -20
    if softcap and softcap <= 256 and q.dtype != F32 and out_dtype != F32:
        p_eps += softcap * 2.0 ** -21
    for b in range(q.shape[0]):
        n = max(0, int(lens[b]))
        k, v = k4.gather(codes, held, cache, layer, ids[b], n)
        want = po.attend(q[b], k, v, scale, softcap)
        # the magnitude of a value is its largest term's: offsets and codes cancel
        room = po.tolerance(q[b], k, v, scale, p_eps, EPS[out_dtype], want)
        if n:
            terms = 2 * float(held[ids[b].long()[: -(-n // cache.block_seq_stride)], layer].abs().max()) * 16
            top = float(q[b].double().abs().sum(-1).max()) * terms * abs(scale)
            room = room + terms * (p_eps + top * (q.shape[-1] + 16) * 2.0 ** -23) + FLOOR[out_dtype]
        off = (got[b].cpu().double() - want).abs()
        assert (off - room).max() <= 0, (float(off.max()), float((off - room).max()))
        if want.norm() > 0:
            most = math.sqrt(3 * p_eps ** 2 + EPS[out_dtype] ** 2) / math.sqrt(3) + 2.0 ** -18
            assert float(off.norm() / want.norm()) <= most, float(off.norm() / want.norm())
    return got


@pytest.mark.parametrize("io", [BF, HF, F32])
@pytest.mark.parametrize("heads,kvh,hd,stride,new", [(8, 2, 128, 32, 1), (16, 2, 64, 16, 1), (8, 1, 128, 16, 1), (4, 4, 64, 7, 1),
                                                     (8, 2, 128, 32, 5), (12, 2, 128, 32, 3), (4, 2, 64, 16, 16), (34, 2, 64, 5, 1),
                                                     (6, 2, 128, 48, 2)])
def test_attend(io, heads, kvh, hd, stride, new):
    gen = torch.Generator().manual_seed(heads + new)
    cache = _cache(kvh, hd, stride)
    lens = torch.tensor([1, 0, 31, 32, 33, 128, 129, 300, 17])
    per = -(-300 // stride)
    ids = _ids(len(lens), per, gen)
    state = k4.fill(cache, len(lens) * per + 2, gen)
    q = torch.randn(len(lens), new, heads, hd, generator=gen).to(io)
    _attend_check(cache, state, ids, lens, q)
    _attend_check(cache, state, ids, lens, q, softcap=20.0, scale=0.3)
    assert _status() == 0


@pytest.mark.parametrize("io,out_dtype", [(BF, HF), (BF, F32), (HF, BF), (F32, BF), (F32, HF)])
def test_attend_output_types(io, out_dtype):
    gen = torch.Generator().manual_seed(4)
    cache = _cache(2, 128, 32)
    ids, lens = _ids(2, 10, gen), torch.tensor([300, 77])
    state = k4.fill(cache, 22, gen)
    _attend_check(cache, state, ids, lens, torch.randn(2, 2, 8, 128, generator=gen).to(io), out_dtype=out_dtype)


@pytest.mark.parametrize("softcap", [0.5, 300.0, 1e4])
@pytest.mark.parametrize("io", [BF, F32])
def test_attend_softcaps(softcap, io):
    gen = torch.Generator().manual_seed(5)
    cache = _cache(2, 64, 16)
    ids, lens = _ids(1, 20, gen), torch.tensor([290])
    state = k4.fill(cache, 22, gen)
    _attend_check(cache, state, ids, lens, torch.randn(1, 1, 8, 64, generator=gen).to(io) * 4, softcap=softcap)


@pytest.mark.parametrize("io", [BF, F32])
@pytest.mark.parametrize("positions,bs", [(5000, 3), (20000, 1)])
def test_attend_long(io, positions, bs):
    gen = torch.Generator().manual_seed(6)
    cache = _cache(2, 64, 32, layers=1)
    per = -(-positions // 32)
    ids = _ids(bs, per, gen)
    state = k4.fill(cache, bs * per + 2, gen)
    lens = torch.tensor([positions - 1000 * b for b in range(bs)])
    for new in (1, 3):
        _attend_check(cache, state, ids, lens, torch.randn(bs, new, 8, 64, generator=gen).to(io), layer=0)


def test_attend_many_sequences():
    gen = torch.Generator().manual_seed(7)
    cache = _cache(1, 64, 16, layers=1)
    lens = torch.randint(-1, 150, (75,), generator=gen)
    ids = _ids(75, 10, gen)
    state = k4.fill(cache, 752, gen)
    _attend_check(cache, state, ids, lens, torch.randn(75, 1, 4, 64, generator=gen).to(BF), layer=0)


def test_attend_values_of_all_sizes():
    """Scales and offsets from 2^-24 to fp16's largest side by side, zero rows, rows of one value."""
    gen = torch.Generator().manual_seed(8)
    cache = _cache(1, 128, 32, layers=1)
    state = k4.fill(cache, 8, gen)
    half = state[1].view(8, 2, 32, 4, 2)
    size = torch.exp2(torch.randint(-18, 8, (8, 2, 32, 1, 1), generator=gen).float())
    half.copy_((half.cpu().float() * size).half())
    half[1, 1, 3] = 0
    half[1, 1, 4, :, 0] = 0
    half[2, 1, 5, 1, 1] = 60000.0
    half[:, 0].mul_(0)                      # K: every position as likely
    half[:, 0, :, :, 1] = 0.5
    ids = torch.arange(8, dtype=torch.int32).view(1, 8)
    for io in (BF, F32):
        for length in (256, 60, 200):
            _attend_check(cache, state, ids, torch.tensor([length]), torch.randn(1, 1, 4, 128, generator=gen).to(io), layer=0)


def test_attend_bad_rows_show_where_they_are_seen():
    """NaN in the scales of dead positions changes nothing; in a live one the rows that see it, in all elements or none."""
    gen = torch.Generator().manual_seed(9)
    cache = _cache(2, 64, 16, layers=1)
    state = k4.fill(cache, 12, gen)
    ids = _ids(1, 10, gen)
    q = torch.randn(1, 4, 4, 64, generator=gen).to(BF)
    call = lambda n: _attention().kv_attend(q.cuda(), cache, state, block_index=0, seq_block_ids=ids.cuda(), seq_lens=torch.tensor([n]).cuda())
    want = call(100)
    half = state[1].view(12, 2, 2, 16, 2, 2)
    for slot in (0, 1):
        for value in (math.nan, math.inf):
            was = half.clone()
            half[int(ids[0, 6]), :, slot, 4] = value                     # position 100: behind the length
            assert torch.equal(call(100), want)
            half.copy_(was)
            half[int(ids[0, 6]), 0, slot, 1] = value                     # position 97: tokens 1 .. 3 see it, head 0
            got = call(100)
            assert torch.equal(got[:, 0], want[:, 0]) and torch.equal(got[:, :, 2:], want[:, :, 2:])
            assert torch.isnan(got[:, 1:, :2]).all()
            half.copy_(was)


def test_captured_and_replayed():
    """Write and attention of a step in one graph, replayed with other positions; two graphs on two streams."""
    A = _attention()
    made = []
    for seed in (1, 2):
        gen = torch.Generator().manual_seed(seed)
        cache = _cache(2, 128, 16)
        ids = _ids(3, 20, gen).cuda()
        state = k4.fill(cache, 62, gen)
        qkv = torch.randn(3, 1, 12 * 128, generator=gen).to(BF).cuda()
        pos = torch.tensor([10, 200, 70], dtype=torch.int32).cuda()
        freqs = _freqs(128).cuda()

        def step(qkv=qkv, pos=pos, state=state, ids=ids, cache=cache, freqs=freqs):
            q, k, v = (p.unflatten(-1, (-1, 128)) for p in qkv.split([8 * 128, 256, 256], dim=-1))
            q, k = A.norm_rope_kv_write(q, k, v, cache, state, block_index=0, seq_block_ids=ids, start_positions=pos, freqs=freqs)
            return A.kv_attend(q, cache, state, block_index=0, seq_block_ids=ids, seq_lens=pos + 1)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        made.append((graph, step, state, pos, qkv, out))
    streams = [torch.cuda.Stream() for _ in made]
    for n in range(4):
        for graph, step, state, pos, qkv, out in made:
            pos.add_(1)
            qkv.mul_(-1.1)
        torch.cuda.synchronize()
        ref = [([t.clone() for t in m[2]], m) for m in made]
        for s, m in zip(streams, made):
            with torch.cuda.stream(s):
                m[0].replay()
        torch.cuda.synchronize()
        for before, (graph, step, state, pos, qkv, out) in ref:
            after = [t.clone() for t in state]
            for t, b in zip(state, before):
                t.copy_(b)
            assert torch.equal(step(), out) and all(torch.equal(a, b) for a, b in zip(after, state))


def test_rows_and_pages_beyond_32_bits_of_bytes():
    """A slab of more than 4 GB, its last pages."""
    A = _attention()
    cache = _cache(8, 128, 64, layers=8)       # 512 KB of codes and 128 KB of scales a page
    pages = 9000
    state = cache.allocate(pages)
    gen = torch.Generator().manual_seed(10)
    ids = torch.tensor([[pages - 1, 8200, 1]], dtype=torch.int32)
    k, v = (torch.randn(1, 150, 8, 128, generator=gen).to(BF) for _ in range(2))
    zero = torch.zeros(1, dtype=torch.int32)
    q, _ = _write(cache, state, ids, zero, torch.randn(1, 150, 16, 128, generator=gen).to(BF).cuda(), k.cuda(), v.cuda(), layer=7)
    kk, vv = A.kv_read(cache, state, block_index=7, seq_block_ids=ids.cuda(), seq_lens=torch.tensor([150]).cuda(), max_seq_len=150, dtype=F32)
    held = k4.scales_of(v)
    want = k4.values(k4.to_code(k4.quotients(v, held)), held)
    assert (vv.cpu().double() - want).abs().max() < 1e-5
    got = A.kv_attend(q[:, -1:], cache, state, block_index=7, seq_block_ids=ids.cuda(), seq_lens=torch.tensor([150]).cuda(), out_dtype=F32)
    ref = ko.attend(q[0, -1:].cpu(), kk[0].cpu().double(), vv[0].cpu().double(), [150], 128 ** -0.5)
    assert (got[0].cpu().double() - ref).abs().max() < 1e-5
    assert _status() == 0


# ---------------------------------------------------------------------- together
@pytest.mark.parametrize("io", [BF, F32])
def test_prompt_continuation_and_steps_together(io):
    """A serving loop's calls: a padded batch of prompts written and attended, a continued one over
    what the cache holds, and single tokens."""
    A = _attention()
    gen = torch.Generator().manual_seed(11)
    heads, kvh, hd, stride = 8, 2, 64, 16
    cache = _cache(kvh, hd, stride)
    state = cache.allocate(40)
    ids = _ids(2, 12, gen)
    kw = dict(block_index=1, seq_block_ids=ids.cuda())
    lens = torch.tensor([45, 70])

    def rows(sl):
        qkv = torch.randn(2, sl, (heads + 2 * kvh) * hd, generator=gen).to(io).cuda()
        return [p.unflatten(-1, (-1, hd)) for p in qkv.split([heads * hd, kvh * hd, kvh * hd], dim=-1)]

    q, k, v = rows(70)
    rq, rk = _write(cache, state, ids, torch.zeros(2, dtype=torch.int32), q, k, v, lens=lens)
    # the padded batch without its padding
    take = torch.cat([torch.arange(45), 70 + torch.arange(70)]).cuda()
    pq, pk, pv = (t.reshape(140, -1, hd)[take] for t in (rq, rk, v))
    cu = torch.tensor([0, 45, 115]).cuda()
    got = A.prompt_attend(pq, pk, pv, cu_seqlens=cu)
    want, room = po.packed(pq.cpu(), pk.cpu(), pv.cpu(), cu, cu, hd ** -0.5, None, 0 if io == F32 else EPS[io], EPS[io])
    assert ((got.cpu().double() - want).abs() - room).max() <= 0
    # ten more tokens each: the cached positions, then the new ones
    q, k, v = rows(10)
    rq, rk = _write(cache, state, ids, lens, q, k, v)
    kc, vc = A.kv_read(cache, state, seq_lens=lens.cuda(), max_seq_len=70, dtype=io, **kw)
    kk, vv = (torch.cat([c[0, :45], n[0], c[1, :70], n[1]]) for c, n in ((kc, rk), (vc, v)))
    cu, cu_k = torch.tensor([0, 10, 20]).cuda(), torch.tensor([0, 55, 135]).cuda()
    flat = rq.reshape(20, heads, hd)
    got = A.prompt_attend(flat, kk, vv, cu_seqlens=cu, cu_seqlens_k=cu_k)
    want, room = po.packed(flat.cpu(), kk.cpu(), vv.cpu(), cu, cu_k, hd ** -0.5, None, 0 if io == F32 else EPS[io], EPS[io])
    assert ((got.cpu().double() - want).abs() - room).max() <= 0
    lens = lens + 10
    for _ in range(3):
        q, k, v = rows(1)
        rq, rk = _write(cache, state, ids, lens, q, k, v)
        lens = lens + 1
        _attend_check(cache, state, ids, lens, rq.cpu())
    assert _status() == 0
