"""Attention of whole prompts at the ends of its range, against its definition in 64 bits."""
import math

import pytest
import torch

import test_gpu_prompt as base
from oracle import prompt_oracle as po

pytestmark = pytest.mark.gpu

BF, HF, F32, EPS = base.BF, base.HF, base.F32, base.EPS


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("softcap", [300.0, 884.0, 1250.0, 1e4, 1e5, 1e6, 1e7, 1e8, 1e12, 3.4e38])
def test_large_softcaps(softcap, hd, dtype):
    """Ordinary scores far below the cap: as without one, in the largest error and in the 2-norm.
    The cap's own error is 2^-20.8 of a score at most, of scores up to 16 and twice in a weight:
    within 2^-15."""
    for lens, lens_k in (([190, 33], None), ([40], [3000])):
        q, k, v, cu, cu_k = base._inputs(lens, lens_k, 4, 2, hd, dtype, seed=int(math.log(softcap)))
        got = base._call(q, k, v, cu, cu_k, softcap=softcap)
        p_eps = 0.0 if dtype == F32 else EPS[dtype]
        want, room = po.packed(q, k, v, cu, cu_k, hd ** -0.5, softcap, p_eps, EPS[dtype])
        off = (got.cpu().double() - want).abs()
        assert (off - room).max() <= 0, float(off.max())
        assert float(off.norm() / want.norm()) <= math.sqrt(p_eps ** 2 + EPS[dtype] ** 2) / math.sqrt(3) + 2.0 ** -15
    assert base._status() == 0


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("softcap", [200.0, 400.0, 3000.0, 1e5])
def test_scores_near_large_softcaps(softcap, dtype):
    """Scores of a part of the cap up to several caps, which only the keys' last tiles have; q and k
    along one direction, so that a score's terms are of one sign.  A score S of 32 bits is off by
    (hd + 8) 2^-23 S, its capped value by as much of its slope, sech^2, and by 2^-20 of the cap's
    magnitude where it is computed apart from its neighbours': the weights of two scores near each
    other differ by that at most.  The values are of one sign and of one size, so that the output
    is off by half a step and by what the weights are."""
    hd, n = 64, 400
    g = torch.Generator().manual_seed(3)
    sign = torch.randint(0, 2, (hd,), generator=g) * 2.0 - 1
    q = (sign * 4).repeat(n, 2, 1).to(dtype)
    top = 3 * softcap / (hd * 4 / 8)
    size = torch.cat([torch.zeros(200), torch.linspace(0, top, 200)])
    k = (sign * size[:, None, None]).repeat(1, 1, 1).to(dtype)
    v = (1 + torch.rand(n, 1, hd, generator=g)).to(dtype)
    cu = torch.tensor([0, n])
    got = base._call(q, k, v, cu, softcap=softcap)
    want = po.attend(q, k, v, hd ** -0.5, softcap)
    off = (got.cpu().double() - want).abs()
    # the largest slope times S is c z sech^2(z) <= 0.45 c
    weight = 2 * softcap * (0.45 * (hd + 8) * 2.0 ** -23 + 2.0 ** -20)
    p_eps = 0.0 if dtype == F32 else EPS[dtype]
    assert (off - want.abs() * (p_eps + EPS[dtype] + min(weight, 1.0) + 2.0 ** -18)).max() <= 0


@pytest.mark.parametrize("where", [0, 130, 500])
@pytest.mark.parametrize("lens,lens_k", [([700], [700]), ([60], [4000]), ([3, 200], [1000, 900])], ids=str)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_an_output_of_small_weights(dtype, lens, lens_k, where):
    """One key has nearly all of the weight and a value of zero: the output is that of weights of
    2^-18 to 2^-24 of it, each to half a step of the type of v.  All terms of a score have one
    sign, scores are up to 15, and a weight is off by twice a score's error at most."""
    hd = 64
    g = torch.Generator().manual_seed(where + sum(lens))
    cu, cu_k = base._cu(lens), base._cu(lens_k)
    q = torch.ones(int(cu[-1]), 4, hd, dtype=dtype)
    k = ((torch.rand(int(cu_k[-1]), 2, 1, generator=g) * 4 - 2) / 8).expand(-1, -1, hd).to(dtype).contiguous()
    v = (0.5 + torch.rand(int(cu_k[-1]), 2, hd, generator=g)).to(dtype)
    for b in range(len(lens)):
        k[int(cu_k[b]) + where], v[int(cu_k[b]) + where] = 14.5 / 8, 0.0
    got = base._call(q, k, v, cu, cu_k, out_dtype=F32)
    want, _ = po.packed(q, k, v, cu, cu_k, hd ** -0.5)
    p_eps = 0.0 if dtype == F32 else EPS[dtype]
    room = want.abs() * (p_eps + 2.0 ** -24 + 2 * 16 * (hd + 8) * 2.0 ** -23 + 2.0 ** -18)
    off = (got.cpu().double() - want).abs()
    assert (off - room).max() <= 0, float((off / want.clamp(min=1e-30)).max())


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("at", [3, 150, 290])
def test_bad_values_of_weights_below_32_bits(dtype, bad, at):
    """An infinity or NaN in the values of a key whose weight is 2^-400 shows in every row that sees it (as
    an infinity or as NaN), wherever it lies among the tiles and parts, and in no other."""
    hd = 64
    g = torch.Generator().manual_seed(at)
    for lens, lens_k in (([300], [300]), ([40], [2000])):
        cu, cu_k = base._cu(lens), base._cu(lens_k)
        n, m = lens[0], lens_k[0]
        q = torch.ones(n, 2, hd, dtype=dtype)
        k = ((torch.rand(m, 1, 1, generator=g) * 2 - 1) / 8).expand(-1, -1, hd).to(dtype).contiguous()
        v = torch.randn(m, 1, hd, generator=g).to(dtype)
        k[at] = -280.0 / 8
        clean = base._call(q, k, v, cu, cu_k).cpu()
        v[at, 0, 7] = bad
        got = base._call(q, k, v, cu, cu_k).cpu()
        sees = torch.arange(n) + m - n >= at
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[sees, :, 7] = True
        assert torch.equal(got[~hit], clean[~hit])
        assert not torch.isfinite(got[hit]).any()
        if math.isnan(bad):
            assert torch.isnan(got[hit]).all()


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_an_infinite_value_before_scores_that_outgrow_it(dtype):
    """The running sums have an infinity when a maximum 2^400 above comes."""
    hd = 64
    g = torch.Generator().manual_seed(1)
    q = torch.ones(600, 2, hd, dtype=dtype)
    k = ((torch.rand(600, 1, 1, generator=g) * 2 - 1) / 8).expand(-1, -1, hd).to(dtype).contiguous()
    v = torch.randn(600, 1, hd, generator=g).to(dtype)
    k[420] = 280.0 / 8
    v[5, 0, 9] = math.inf
    cu = torch.tensor([0, 600])
    got = base._call(q, k, v, cu).cpu()
    assert torch.isfinite(got[:5]).all() and not torch.isfinite(got[5:, :, 9]).any()
    assert torch.isfinite(got[..., torch.arange(hd) != 9]).all()
