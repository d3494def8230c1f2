"""Which masks count as the causal one: every form and every other entry, on the GPU."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")


def _causal(mask, bs=2, new_lens=None):
    """Whether the mask passes."""
    from shark_platform_b200 import attention as A, moe

    assert moe.device_status() == 0
    A._check_causal(mask.cuda() if mask.device.type == "cpu" else mask, bs, new_lens, torch.device("cuda", 0))
    try:
        return moe.device_status() == 0
    except moe.C.B200MoeError as e:
        assert "status word = 2" in str(e)
        return False


def _mask(sl, first=0, lens=None, low=-INF, rows=False):
    unseen = torch.ones(sl, first + sl, dtype=torch.bool).triu(first + 1)[None, None]
    if lens is not None:
        n = torch.tensor(lens)[:, None]
        unseen = unseen | (torch.arange(first + sl)[None] >= first + n)[:, None, None]
        if rows:
            unseen = unseen | (torch.arange(sl)[None] >= n)[:, None, :, None]
    return torch.zeros(unseen.shape, dtype=torch.float64).masked_fill(unseen, low)


@pytest.mark.parametrize("sl,first", [(1, 0), (2, 0), (7, 0), (1, 5), (7, 5), (64, 0), (255, 1), (256, 0), (257, 3), (600, 8), (1030, 0)])
@pytest.mark.parametrize("low,dtype", [(-INF, torch.float32), (-1e4, torch.bfloat16), (-65504.0, torch.float16), (-1e300, torch.float64)])
def test_causal_masks(sl, first, low, dtype):
    for lens, rows in itertools.product((None, [sl, sl], [sl, 0], [sl // 2, sl], [1, sl - 1]), (False, True)):
        m = _mask(sl, first, lens, max(low, torch.finfo(dtype).min) if low > -INF else low, rows).to(dtype)
        for form in (m, m[-1, 0], m[:1, 0], m.expand(-1, 3, -1, -1), m.to(torch.float64).repeat(1, 3, 1, 1), m == 0):
            assert _causal(form)
    wide = torch.full((2, 1, sl, first + sl + 3), float("nan"), dtype=dtype, device="cuda")  # rows that are not 16 bytes apart
    wide[..., 1:-2] = _mask(sl, first, None, max(low, torch.finfo(dtype).min) if low > -INF else low).to(dtype)
    assert _causal(wide[..., 1:-2])
    t = _mask(sl, first).cuda().transpose(-1, -2).contiguous().transpose(-1, -2)
    assert _causal(t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first", [0, 5])
def test_any_other_entry(first, dtype):
    """One entry changed in a row of tokens: seen or not, or neither."""
    sl = 6
    for i, j in itertools.product(range(sl), range(first + sl)):
        m = _mask(sl, first, [sl, 4]).to(dtype)
        was = m[0, 0, i, j].item()
        m[0, 0, i, j] = -INF if j <= first + i else 0.0
        if (i, j) != (sl - 1, first + sl - 1):  # without its last entry it is the mask of a token less
            assert not _causal(m) and not _causal(m == 0) and not _causal(m[0, 0])
        else:
            assert _causal(m)
        for value in (-3.0, 1.0, INF, float("nan")):
            m[0, 0, i, j] = value
            assert not _causal(m)
        m[0, 0, i, j] = was
        assert _causal(m)


@pytest.mark.parametrize("first", [0, 5])
def test_rows_of_padding(first):
    """They may see any of the tokens, and nothing behind them."""
    m = _mask(6, first, [6, 4])
    m[1, 0, 4:] = -INF
    m[1, 0, 5, first + 3] = 0.0
    m[1, 0, 4, 0] = -0.7
    assert _causal(m)
    m[1, 0, 4, first + 5] = 0.0
    assert not _causal(m)


def test_tokens_by_new_lens():
    lens = lambda *n: torch.tensor(n)
    m = _mask(6, 0, [6, 4])
    assert _causal(m, new_lens=lens(6, 4)) and _causal(m, new_lens=lens(3, -1)) and _causal(m.expand(-1, 2, -1, -1), new_lens=lens(6, 4))
    assert not _causal(m, new_lens=lens(6, 5)) and not _causal(m[1, 0], new_lens=lens(3, 5)) and not _causal(m.repeat(1, 3, 1, 1), new_lens=lens(0, 6))
    assert _causal(_mask(6), new_lens=lens(6, 5)) and _causal(_mask(6), new_lens=lens(600, 5))


@pytest.mark.parametrize("sl", [300, 700])
def test_other_masks_of_many_rows(sl):
    """More rows than are sampled: windows, chunks, strictly earlier positions, holes beside the samples."""
    i, j = torch.arange(sl)[:, None], torch.arange(sl)[None]
    c = _mask(sl)[0, 0]
    others = [c.masked_fill(j < i - 100, -INF), c.masked_fill(j // 128 < i // 128, -INF), c.masked_fill(j == i, -INF), torch.zeros(sl, sl, dtype=c.dtype),
              c.masked_fill(j < 5, 0.0), c.masked_fill(j < 3, -INF), torch.full_like(c, -INF).masked_fill_(j < i, 0.0),
              c.masked_fill((i >= 100) & (i < 200), -INF), c.masked_fill((j == sl - 1), 0.0), c - 0.1 * (i - j).abs()]
    for at in (0, 1, 2, 3, 255, 256, sl - 2):
        others.append(c.index_put((torch.tensor([at]), torch.tensor([at])), torch.tensor(-INF, dtype=c.dtype)))
        others.append(c.index_put((torch.tensor([at]), torch.tensor([at + 1])), torch.tensor(0.0, dtype=c.dtype)))
    for m in others:
        assert not _causal(m) and not _causal(torch.stack([c, m])[:, None])
    assert _causal(torch.full((sl, sl), -INF))  # no tokens


def test_many_masks():
    m = _mask(3, 2).expand(70000, 1, 3, 5).clone()
    assert _causal(m, 70000)
    m[69999, 0, 1, 0] = -1.0
    assert not _causal(m, 70000)
