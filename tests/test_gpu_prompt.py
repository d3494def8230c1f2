"""Attention of whole prompts on the GPU against its definition in 64 bits."""
import math

import pytest
import torch

from oracle import prompt_oracle as po

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
# half a step of each type, relative
EPS = {F32: 2.0 ** -24, HF: 2.0 ** -11, BF: 2.0 ** -8}


def _attention():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    from shark_platform_b200 import attention as A

    return A


def _status():
    from shark_platform_b200 import moe

    return moe.device_status()


def _cu(lens, first=0):
    return torch.tensor([first] + (first + torch.tensor(lens, dtype=torch.long).cumsum(0)).tolist())


def _inputs(lens, lens_k, heads, kvh, hd, dtype, seed=0, before=0, behind=0, std=1.5):
    g = torch.Generator().manual_seed(seed)
    cu, cu_k = _cu(lens, before), _cu(lens_k if lens_k is not None else lens, before)
    q = (torch.randn(int(cu[-1]) + behind, heads, hd, generator=g) * std).to(dtype)
    k, v = (torch.randn(int(cu_k[-1]) + behind, kvh, hd, generator=g).to(dtype) for _ in range(2))
    return q, k, v, cu, cu_k


def _call(q, k, v, cu, cu_k=None, **kw):
    return _attention().prompt_attend(q.cuda(), k.cuda(), v.cuda(), cu_seqlens=cu.cuda(),
                                      cu_seqlens_k=None if cu_k is None else cu_k.cuda(), **kw)


def _check(got, q, k, v, cu, cu_k, scale=None, softcap=None, out_dtype=None):
    out_dtype = out_dtype or q.dtype
    scale = scale or 1 / math.sqrt(q.shape[-1])
    assert got.dtype == out_dtype and got.shape == q.shape and got.is_contiguous()
    # probabilities are rounded to the type of v, 32-bit ones not at all
    want, room = po.packed(q, k, v, cu, cu_k, scale, softcap, 0.0 if q.dtype == F32 else EPS[q.dtype], EPS[out_dtype])
    off = (got.cpu().double() - want).abs()
    assert (off - room).max() <= 0, (float(off.max()), float((off - room).max()))
    live = want.norm()
    if live > 0 and q.dtype != F32:
        # in the 2-norm: two independent roundings, at most eps / sqrt(3) in the mean square each
        # (an output of other bits has its own)
        most = math.sqrt(EPS[q.dtype] ** 2 + EPS[out_dtype] ** 2) / math.sqrt(3)
        assert float(off.norm() / live) <= most + 2.0 ** -18
    return want


LENS = [[1], [2], [17], [63, 1, 64, 65], [127, 128, 129], [255, 3, 257], [0, 5, 0, 300, 1], [640]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_lengths(lens, dtype):
    q, k, v, cu, cu_k = _inputs(lens, None, 8, 2, 128, dtype, seed=sum(lens))
    _check(_call(q, k, v, cu), q, k, v, cu, cu_k)
    assert _status() == 0


@pytest.mark.parametrize("heads,kvh", [(1, 1), (4, 4), (2, 1), (3, 1), (12, 2), (16, 2), (64, 1), (96, 1), (130, 1), (200, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_heads(heads, kvh, hd):
    """Groups of heads that fill a tile, leave rows over, take a token each or several tiles a token."""
    for dtype in (BF, F32):
        q, k, v, cu, cu_k = _inputs([70, 133], None, heads, kvh, hd, dtype, seed=heads)
        _check(_call(q, k, v, cu), q, k, v, cu, cu_k)


@pytest.mark.parametrize("lens,lens_k", [([1], [1000]), ([5, 1, 40], [5, 700, 300]), ([130], [515]), ([16, 16], [128, 129]),
                                         ([64], [2000]), ([3, 3], [0, 4]), ([300], [301])], ids=str)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_continued(lens, lens_k, dtype):
    """More keys than queries: the cached positions before the prompt."""
    q, k, v, cu, cu_k = _inputs(lens, lens_k, 8, 2, 64, dtype, seed=7)
    _check(_call(q, k, v, cu, cu_k), q, k, v, cu, cu_k)
    assert _status() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_that_see_nothing(dtype):
    """More queries than keys: the first rows attend nothing and are zero."""
    q, k, v, cu, cu_k = _inputs([200, 10, 150], [60, 0, 149], 4, 2, 128, dtype)
    got = _call(q, k, v, cu, cu_k)
    _check(got, q, k, v, cu, cu_k)
    assert not got[:140].any() and not got[200:210].any() and not got[210].any() and got[211].any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_no_sequence(dtype):
    """In front of the first and behind the last sequence: zeros, whatever q, k and v hold there."""
    q, k, v, cu, cu_k = _inputs([33, 90], None, 4, 1, 64, dtype, before=5, behind=77)
    for t in (q, k, v):
        t[:5], t[-77:] = math.nan, math.inf
    got = _call(q, k, v, cu)
    assert torch.isfinite(got).all() and not got[:5].any() and not got[-77:].any()
    z = [t.clone() for t in (q, k, v)]
    for t in z:
        t[:5], t[-77:] = 0, 0
    _check(got, *z, cu, cu_k)


@pytest.mark.parametrize("dtype,out_dtype", [(BF, F32), (BF, HF), (HF, BF), (HF, F32), (F32, HF), (F32, BF)])
def test_output_types(dtype, out_dtype):
    q, k, v, cu, cu_k = _inputs([150, 20], None, 4, 2, 128, dtype)
    _check(_call(q, k, v, cu, out_dtype=out_dtype), q, k, v, cu, cu_k, out_dtype=out_dtype)


@pytest.mark.parametrize("softcap", [0.5, 30.0, 2000.0])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_softcap_and_scale(softcap, dtype):
    q, k, v, cu, cu_k = _inputs([190], None, 4, 2, 128, dtype, std=8.0)
    _check(_call(q, k, v, cu, softcap=softcap, scale=0.2), q, k, v, cu, cu_k, scale=0.2, softcap=softcap)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_large_scores(dtype):
    """Softmaxes with one position each, rising and falling maxima."""
    q, k, v, cu, cu_k = _inputs([300], None, 2, 1, 64, dtype, std=1.0)
    k = (k.float() * torch.linspace(0.1, 30, 300)[:, None, None]).to(dtype)
    _check(_call(q, k, v, cu), q, k, v, cu, cu_k)
    k = k.flip(0)
    _check(_call(q, k, v, cu), q, k, v, cu, cu_k)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_views(dtype):
    """Views of a fused projection; views that are not aligned to 16 bytes and transposed ones are copied."""
    g = torch.Generator().manual_seed(3)
    heads, kvh, hd, n = 8, 2, 64, 150
    qkv = torch.randn(n, (heads + 2 * kvh) * hd + 8, generator=g).to(dtype).cuda()
    cu = torch.tensor([0, 100, 150]).cuda()
    for at in (0, 8, 3):
        q, k, v = (x.unflatten(-1, (-1, hd)) for x in qkv[:, at:].split([heads * hd, kvh * hd, kvh * hd, 8 - at], dim=-1)[:3])
        got = _attention().prompt_attend(q, k, v, cu_seqlens=cu)
        assert torch.equal(got, _attention().prompt_attend(q.contiguous(), k.contiguous(), v.contiguous(), cu_seqlens=cu))
        _check(got, q.cpu(), k.cpu(), v.cpu(), cu.cpu(), cu.cpu())
    t = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(got, _attention().prompt_attend(*t, cu_seqlens=cu.to(torch.int32)))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_bad_values_show_in_the_rows_that_attend_them(dtype, bad):
    """A bad value of k or v in the middle of a tile: earlier rows and other sequences do not see it."""
    q, k, v, cu, cu_k = _inputs([200, 150, 90], None, 4, 2, 64, dtype)
    clean = _call(q, k, v, cu).cpu()
    for which in (k, v):
        at = 200 + 77
        was = which[at].clone()
        which[at, 1, 5] = bad
        got = _call(q, k, v, cu).cpu()
        assert torch.equal(got[:at], clean[:at]) and torch.equal(got[350:], clean[350:])
        assert torch.equal(got[at:350, :2], clean[at:350, :2])  # the other kv head's
        if which is v:
            want = po.attend(q[200:350, 2:], k[200:350, 1:], v[200:350, 1:], 1 / 8)
            hit = got[200:350, 2:].double()
            assert torch.equal(torch.isnan(hit), torch.isnan(want)) and torch.equal(torch.isinf(hit), torch.isinf(want))
            assert torch.equal(hit[torch.isinf(hit)], want[torch.isinf(want)])
            keep = torch.arange(64) != 5
            assert torch.equal(got[at:350, 2:][..., keep], clean[at:350, 2:][..., keep])
        which[at] = was
    # and in a tile that all rows of a later tile see whole
    v[3, 0, 9] = bad
    got = _call(q, k, v, cu).cpu()
    assert torch.equal(got[:3], clean[:3]) and not torch.isfinite(got[3:200, :2, 9]).any()
    assert torch.equal(got[200:], clean[200:])


def test_many_sequences():
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 40, (150,), generator=g).tolist()
    for dtype in (BF, F32):
        q, k, v, cu, cu_k = _inputs(lens, None, 4, 2, 64, dtype, seed=6)
        _check(_call(q, k, v, cu), q, k, v, cu, cu_k)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_thousands_of_sequences(dtype):
    """More sequences than a warp looks at in one go, at one and at several places of the list."""
    g = torch.Generator().manual_seed(15)
    lens = torch.randint(0, 4, (3500,), generator=g)
    lens[1234], lens[3400] = 200, 131
    q, k, v, cu, cu_k = _inputs(lens.tolist(), None, 4, 2, 64, dtype, seed=16)
    _check(_call(q, k, v, cu), q, k, v, cu, cu_k)


@pytest.mark.parametrize("dtype,rows", [(BF, 300000), (F32, 150000)])
def test_rows_beyond_32_bits_of_elements(dtype, rows):
    """q of more than 2^32 bytes, k and v rows of a tensor of more than 2^32 bytes: the last sequences."""
    q, k, v, cu, _ = _inputs([100, 100], None, 64, 1, 128, dtype, seed=18)
    full = torch.zeros(rows, 64, 128, dtype=dtype, device="cuda")
    wide = torch.zeros(rows, 16384, dtype=dtype, device="cuda")
    kk, vv = (wide[:, at:at + 128].unflatten(1, (1, 128)) for at in (128, 16000))
    for to, x in ((full, q), (kk, k), (vv, v)):
        to[-200:] = x.cuda()
    got = _call(full, kk, vv, torch.arange(0, rows + 1, 100))
    _check(got[-200:], q, k, v, cu, cu)
    assert got[:-200].abs().max() == 0


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("scale,softcap", [(-0.125, None), (-0.125, 20.0), (0.0, None), (0.0, 20.0), (1e-6, 0.1), (40.0, 0.01)])
def test_scales_of_any_sign_and_size(dtype, scale, softcap):
    q, k, v, cu, cu_k = _inputs([150, 20], None, 4, 2, 64, dtype, seed=17)
    got = _call(q, k, v, cu, scale=scale, softcap=softcap)
    want, room = po.packed(q, k, v, cu, cu_k, scale, softcap, 0.0 if dtype == F32 else EPS[dtype], EPS[dtype])
    assert ((got.cpu().double() - want).abs() - room).max() <= 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_longer(dtype):
    """More items than SMs, several tiles of keys: the list of items and the rings go round."""
    lens = [1300, 900, 2050]
    q, k, v, cu, cu_k = _inputs(lens, None, 8, 2, 128, dtype, seed=9)
    _check(_call(q, k, v, cu), q, k, v, cu, cu_k)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (6, 1, 64), (130, 1, 64)])
@pytest.mark.parametrize("lens,lens_k", [([1], [6000]), ([5, 90, 1, 0, 33], [5, 4000, 1, 700, 6500]), ([64, 2], [3500, 0]),
                                         ([300], [2500]), ([40, 7], [20, 5000])], ids=str)
def test_split_keys(lens, lens_k, heads, kvh, hd, dtype):
    """Few rows, long keys: parts of the keys of a tile in several CTAs, joined; sequences of other lengths beside them."""
    q, k, v, cu, cu_k = _inputs(lens, lens_k, heads, kvh, hd, dtype, seed=12, behind=3)
    q[-3:], k[-3:], v[-3:] = math.nan, math.nan, math.nan
    got = _call(q, k, v, cu, cu_k)
    assert not got[-3:].any()
    for t in (q, k, v):
        t[-3:] = 0
    _check(got, q, k, v, cu, cu_k)
    _check(_call(q, k, v, cu, cu_k, softcap=30.0, out_dtype=F32), q, k, v, cu, cu_k, softcap=30.0, out_dtype=F32)
    assert _status() == 0


@pytest.mark.parametrize("lens,before,heads,kvh", [
    ([3] * 16, [300] * 15 + [5000], 8, 8), ([3] * 16, [1100] * 16, 8, 8),          # one part each by the mean
    ([16] * 8, [8000, 500, 200, 4000, 0, 900, 300, 2000], 4, 2), ([1] * 32, list(range(0, 3200, 100)), 4, 1),
    ([1] * 40, [2000] + [700] * 39, 4, 1),                                          # more sequences than lanes
    ([70, 0, 5], [3000, 3000, 9000], 4, 2), ([1, 0, 0, 0], [9000, 0, 100, 0], 2, 2)], ids=str)
def test_split_keys_of_uneven_sequences(lens, before, heads, kvh):
    lens_k = [n + m for n, m in zip(lens, before)]
    for dtype, softcap in ((BF, None), (HF, 20.0)):
        q, k, v, cu, cu_k = _inputs(lens, lens_k, heads, kvh, 64, dtype, seed=19)
        got = _call(q, k, v, cu, cu_k, softcap=softcap)
        _check(got, q, k, v, cu, cu_k, softcap=softcap)
        assert torch.equal(got, _call(q, k, v, cu, cu_k, softcap=softcap))
    assert _status() == 0


def test_split_keys_with_bad_values():
    """An infinity in one part and a NaN in another: the rows that attend them."""
    q, k, v, cu, cu_k = _inputs([60], [5000], 8, 2, 128, BF, seed=13)
    clean = _call(q, k, v, cu, cu_k).cpu()
    v[100, 0, 3], v[4980, 1, 7] = math.inf, math.nan
    got = _call(q, k, v, cu, cu_k).cpu()
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[:, :4, 3] = True
    hit[40:, 4:, 7] = True  # row i attends keys up to 4940 + i
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any()


def test_nothing():
    A = _attention()
    e = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert A.prompt_attend(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), cu_seqlens=z).shape == (0, 4, 64)
    x = torch.ones(9, 4, 64, dtype=BF, device="cuda")
    assert not A.prompt_attend(x, x, x, cu_seqlens=z).any()
    assert not A.prompt_attend(x, e(0, 4, 64), e(0, 4, 64), cu_seqlens=torch.tensor([0, 9]).cuda(),
                               cu_seqlens_k=torch.tensor([0, 0]).cuda()).any()
    assert _status() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_bounds_that_leave_the_rows(dtype):
    """Sequences are cut to the rows there are, and the status word says so."""
    from shark_platform_b200 import _cabi as C

    q, k, v, cu, cu_k = _inputs([40, 60], None, 4, 2, 64, dtype)
    want = _call(q, k, v, cu).cpu()
    for bad in ([0, 40, 4000], [-7, 40, 100]):
        got = _call(q, k, v, torch.tensor(bad)).cpu()
        assert torch.equal(got, want)
        with pytest.raises(C.B200MoeError, match="status word"):
            _status()
    got = _call(q, k, v, torch.tensor([0, 40, 10, 100]))  # decreasing: the second is empty
    assert got.shape == want.shape and torch.equal(got[:10].cpu(), want[:10])
    with pytest.raises(C.B200MoeError, match="status word"):
        _status()
    assert _status() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_captured_and_replayed(dtype):
    """A captured call reads the bounds and rows of its replay; two graphs at once on two streams."""
    A = _attention()
    made = []
    for seed, lens in ((1, [100, 60]), (2, [30, 130])):
        q, k, v, cu, cu_k = (t.cuda() for t in _inputs(lens, None, 8, 2, 128, dtype, seed=seed))
        A.prompt_attend(q, k, v, cu_seqlens=cu)
        cu = cu.to(torch.int32)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = A.prompt_attend(q, k, v, cu_seqlens=cu)
        made.append((graph, q, k, v, cu, out))
    streams = [torch.cuda.Stream() for _ in made]
    for round_ in range(3):
        for i, (graph, q, k, v, cu, out) in enumerate(made):
            cu.copy_(torch.tensor([0, 20 + 30 * round_ + i, 160], dtype=torch.int32))
            v.mul_(1.5)
        torch.cuda.synchronize()
        for s, m in zip(streams, made):
            with torch.cuda.stream(s):
                for _ in range(3):
                    m[0].replay()
        torch.cuda.synchronize()
        for graph, q, k, v, cu, out in made:
            assert torch.equal(out, A.prompt_attend(q, k, v, cu_seqlens=cu))
            _check(out, *(t.cpu() for t in (q, k, v)), cu.cpu(), cu.cpu())


def test_the_same_each_time():
    for dtype in (BF, F32):
        q, k, v, cu, cu_k = (t.cuda() for t in _inputs([400, 33], [2400, 3000], 8, 2, 128, dtype))
        outs = [_attention().prompt_attend(q, k, v, cu_seqlens=cu, cu_seqlens_k=cu_k) for _ in range(4)]
        assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_its_inputs_stay():
    q, k, v, cu, _ = (t.cuda() for t in _inputs([140, 33], None, 8, 2, 128, BF))
    was = [t.clone() for t in (q, k, v, cu)]
    _attention().prompt_attend(q, k, v, cu_seqlens=cu)
    assert all(torch.equal(a, b) for a, b in zip(was, (q, k, v, cu)))
