"""attention_kernel="b200" in the attention block: masks that are the causal one, masks that are
not, and gradients."""
import pytest
import torch

from test_gpu_kv4_block import Model4
from test_gpu_kv8_block import I8, Model, _near

pytestmark = pytest.mark.gpu

INF = float("inf")


def _model(dtype, act=torch.float32, **kw):
    m = (Model4 if dtype == torch.uint8 else Model)(dtype, act=act, **kw)
    m.block.attention_kernel = "b200"
    return m


def _causal(sl, before=0, lens=None, low=-INF, rows=False, dtype=torch.float32):
    """[1 or 2, 1, sl, before + sl]: what a row does not see is `low`; with lens also padding, in
    the columns and (rows) whole rows."""
    unseen = torch.ones(sl, before + sl, dtype=torch.bool).triu(before + 1)[None, None]
    if lens is not None:
        n = torch.tensor(lens)[:, None]
        pad = torch.arange(before + sl)[None] >= before + n
        unseen = unseen | pad[:, None, None]
        if rows:
            unseen = unseen | (torch.arange(sl)[None] >= n)[:, None, :, None]
    return torch.zeros(unseen.shape, dtype=dtype).masked_fill_(unseen, low).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, I8, torch.uint8])
def test_causal_masks_are_taken(dtype):
    """Any form of the causal mask: infinities or large numbers, one for the batch or one each, with padding."""
    from shark_platform_b200 import moe

    m = _model(dtype)
    h = m.rows(20)
    y = m.call(h, start_index=0)
    masks = [_causal(20), _causal(20)[0, 0], _causal(20, low=-1e9), _causal(20, low=torch.finfo(torch.float16).min, dtype=torch.float16),
             _causal(20, lens=[20, 20]), _causal(20).expand(2, m.heads, 20, 20)]
    for mask in masks:
        assert torch.equal(m.call(h, start_index=0, attention_mask=mask), y)
    for rows in (False, True):
        for lens in ([20, 7], [1, 20], [0, 20]):
            got = m.call(h, start_index=0, attention_mask=_causal(20, lens=lens, rows=rows))
            for b, n in enumerate(lens):
                assert torch.equal(got[b, :n], y[b, :n])
    assert moe.device_status() == 0
    if dtype != torch.float32:
        h = m.rows(9)
        y = m.call(h, start_index=20)
        for mask in (_causal(9), _causal(9, 20), _causal(9, 20, lens=[9, 9]), _causal(9, lens=[9, 9])):
            assert torch.equal(m.call(h, start_index=20, attention_mask=mask), y)
        assert torch.equal(m.call(h, start_index=20, attention_mask=_causal(9, 20, lens=[4, 9]))[0, :4], y[0, :4])
        assert moe.device_status() == 0


def _others(sl, before=0):
    c = _causal(sl, before)[0, 0]
    i, j = torch.arange(sl).cuda()[:, None], torch.arange(before + sl).cuda()[None]
    yield "sliding", c.masked_fill(j < i + before - 3, -INF)
    yield "chunks", c.masked_fill(j // 8 < (i + before) // 8, -INF)
    yield "all seen", torch.zeros_like(c)
    yield "prefix", c.masked_fill(j < before + 5, 0.0)
    yield "one key more", c.index_put((torch.tensor([2]).cuda(), torch.tensor([before + 3]).cuda()), torch.tensor(0.0).cuda())
    yield "one key less", c.index_put((torch.tensor([sl - 2]).cuda(), torch.tensor([2]).cuda()), torch.tensor(-INF).cuda())
    yield "bias", c - 0.25 * (i + before - j).abs()
    yield "padding in front", c.masked_fill(j < 3, -INF)
    yield "nan", c.masked_fill(j == i + before, float("nan"))


@pytest.mark.parametrize("dtype", [torch.float32, I8, torch.uint8])
def test_other_masks_are_reported(dtype):
    """A mask of the right shape that is not the causal one: no silent numbers, the status word says so."""
    from shark_platform_b200 import moe

    m = _model(dtype)
    h = m.rows(20)
    for name, mask in _others(20):
        for form in (mask, torch.stack([_causal(20)[0, 0], mask])[:, None]):  # for the batch, for the second sequence alone
            m.call(h, start_index=0, attention_mask=form)
            with pytest.raises(moe.C.B200MoeError, match="status word"):
                moe.device_status()
    if dtype != torch.float32:
        m.call(m.rows(20), start_index=0)
        for name, mask in _others(9, 20):
            m.call(m.rows(9), start_index=20, attention_mask=mask)
            with pytest.raises(moe.C.B200MoeError, match="status word"):
                moe.device_status()
    assert moe.device_status() == 0


def test_the_tokens_that_new_lens_names_are_looked_at():
    """Rows that the mask leaves out are padding only where new_lens does not call them tokens."""
    from shark_platform_b200 import moe

    m = _model(torch.uint8)
    h = m.rows(20)
    call = lambda lens: m.call(h, start_index=0, attention_mask=_causal(20, lens=[20, 12]), new_lens=torch.tensor(lens).cuda())
    call([20, 12]), call([20, 5])
    assert moe.device_status() == 0
    call([20, 13])
    with pytest.raises(moe.C.B200MoeError, match="status word"):
        moe.device_status()


def test_a_captured_prompt_with_a_mask():
    """The mask of the replay is the one that is looked at."""
    from shark_platform_b200 import moe

    m = _model(torch.uint8)
    h, mask, ids = m.rows(20).cuda(), _causal(20).clone(), m.ids.cuda()
    call = lambda: m.block(h, embedding=m.rope, cache_state=m.state, seq_block_ids=ids, start_index=0, attention_mask=mask)
    y = call().clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, y) and moe.device_status() == 0
    mask[0, 0, 19, 0] = -INF
    graph.replay()
    with pytest.raises(moe.C.B200MoeError, match="status word"):
        moe.device_status()
    mask[0, 0, 19, 0] = 0.0
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, y) and moe.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, I8, torch.uint8])
def test_weights_that_want_gradients(dtype):
    """The prompt attention has no gradient: with weights that want one the call is refused, before the
    cache is written, and taken under no_grad."""
    from shark_platform_b200 import moe

    m = _model(dtype)
    h = m.rows(11)
    with torch.no_grad():
        y = m.call(h, start_index=0)
    m.block._wqkv.requires_grad_()
    before = [t.clone() for t in m.state]
    for t in m.state:
        t.zero_()
    with pytest.raises(moe.C.B200MoeError, match="no gradient"):
        m.call(h, start_index=0)
    assert not any(t.any() for t in m.state)
    with torch.no_grad():
        assert torch.equal(m.call(h, start_index=0), y)
    assert all(torch.equal(a, b) for a, b in zip(m.state, before))
    with torch.inference_mode():
        assert torch.equal(m.call(h, start_index=0), y)
