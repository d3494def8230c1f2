"""B200PagedAttentionBlock with a 4-bit cache and with the packed prompt attention: prompts,
continued prompts, steps of one and of several tokens, against the formulas in 64 bits over the
values that the cache holds."""
import pytest
import torch

from oracle import kv4_oracle as k4
from test_gpu_kv8_block import I8, Model, _near

pytestmark = pytest.mark.gpu


class Model4(Model):
    def held(self, b, n):
        codes, held = k4.page_views(self.state, self.cache)
        return k4.gather(codes, held, self.cache, 1, self.ids[b], n)


@pytest.mark.parametrize("act", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norms,use_hf,softcap,heads,kv_heads", [
    (False, False, None, 4, 2), (True, True, None, 4, 2), (True, False, 30.0, 4, 1), (False, True, 30.0, 12, 1)])
def test_four_bit_block(act, norms, use_hf, softcap, heads, kv_heads):
    from shark_platform_b200 import moe

    m = Model4(torch.uint8, norms, use_hf, softcap, heads, kv_heads, act)
    h = m.rows(20)
    want, new = m.want(h, [0, 0], [0, 0])
    _near(m.call(h, start_index=0), want, act)
    for b in range(2):  # the cache holds what was computed, to half a step of its 32 values' range
        for got, x in zip(m.held(b, 20), new[b]):
            g = k4.groups(x)
            step = ((g.amax(-1) - g.amin(-1)) / 15).repeat_interleave(k4.GROUP, -1)
            # a bf16 block computes x itself to a few half steps of its rows
            assert ((got - x).abs() - 0.51 * step - (1e-3 if act == torch.float32 else 0.05) * x.abs().amax()).max() <= 0
    # the prompt goes on: the cached positions are attended, without a mask and with one
    h = m.rows(13)
    _near(m.call(h, start_index=20), m.want(h, [20, 20], [20, 20])[0], act)
    mask = torch.zeros(2, 1, 7, 7).masked_fill_(torch.ones(7, 7, dtype=torch.bool).triu(1), float("-inf")).cuda()
    h = m.rows(7)
    _near(m.call(h, start_index=33, attention_mask=mask), m.want(h, [33, 33], [33, 33])[0], act)
    # steps: ragged positions, several tokens at once
    at = [40, 36]
    for sl in (1, 1, 4, 16):
        h = m.rows(sl)
        _near(m.call(h, start_positions=torch.tensor(at).cuda()), m.want(h, at)[0], act)
        at = [p + sl for p in at]
    # a padding sequence beside a live one
    h = m.rows(1)
    before = [t.clone() for t in m.state]
    y = m.call(h, start_positions=torch.tensor([at[0], -1]).cuda())
    _near(y[0], m.want(h, [at[0], 0])[0][0], act)
    assert torch.isfinite(y[1]).all()
    pages = m.ids[1].cuda()
    assert all(torch.equal(a[pages].view(torch.uint8), b[pages].view(torch.uint8)) for a, b in zip(m.state, before))
    assert moe.device_status() == 0


@pytest.mark.parametrize("act", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype,softcap,norms", [(torch.float32, None, False), (torch.bfloat16, 30.0, True), (I8, None, True)])
def test_packed_prompt_attention_in_the_block(act, dtype, softcap, norms):
    """attention_kernel="b200": the same block, causal by itself, whether a causal mask comes with the call or not."""
    from shark_platform_b200 import moe

    if not norms and dtype != act:
        pytest.skip("the plain write has one type")
    m = Model(dtype, norms, softcap=softcap, act=act)
    h = m.rows(37)
    m.block.attention_kernel = "b200"
    y = m.call(h, start_index=0)
    _near(y, m.want(h, [0, 0], [0, 0])[0], act)
    mask = torch.zeros(2, 1, 37, 37).masked_fill_(torch.ones(37, 37, dtype=torch.bool).triu(1), float("-inf")).cuda()
    assert torch.equal(m.call(h, start_index=0, attention_mask=mask), y)
    m.block.attention_kernel = "decomposed"
    _near(m.call(h, start_index=0), y.cpu().double(), act)
    if m.cache.quantized:
        m.block.attention_kernel = "b200"
        h = m.rows(9)
        _near(m.call(h, start_index=37), m.want(h, [37, 37], [37, 37])[0], act)
    assert moe.device_status() == 0


def test_padded_prompts_in_the_block():
    """Rows behind a prompt's tokens change none of its rows, whatever they hold."""
    for dtype in (torch.uint8, I8):
        m = (Model4 if dtype == torch.uint8 else Model)(dtype)
        m.block.attention_kernel = "b200"
        h = m.rows(32)
        lens = torch.tensor([32, 19]).cuda()
        y = m.call(h, start_index=0, new_lens=lens)
        h[1, 19:] = 1e4
        again = m.call(h, start_index=0, new_lens=lens)
        assert torch.equal(again[0], y[0]) and torch.equal(again[1, :19], y[1, :19])


@pytest.mark.parametrize("dtype", [torch.uint8, I8])
def test_masks_that_are_not_causal_ones(dtype):
    """A mask of padding alone, or of other lengths, is refused before anything is written."""
    from shark_platform_b200 import moe

    m = (Model4 if dtype == torch.uint8 else Model)(dtype)
    m.block.attention_kernel = "b200"
    before = [t.clone() for t in m.state]
    h = m.rows(20)
    for shape in ((2, 1, 1, 20), (2, 1, 20, 1), (2, 1, 20, 24), (2, 1, 24, 20), (20,)):
        with pytest.raises(moe.C.B200MoeError, match="is causal by itself"):
            m.call(h, start_index=0, attention_mask=torch.zeros(shape).cuda())
    assert all(torch.equal(a, b) for a, b in zip(before, m.state))


def test_patching_takes_the_kernel():
    from shark_platform_b200 import attention as A

    m = Model(I8)

    class Child(torch.nn.Module):
        pass

    child = Child()
    for name in ("theta", "cache", "head_count", "head_dim", "head_count_kv", "block_index"):
        setattr(child, name, getattr(m.block, name))
    child.attn_norm = type("N", (), {"epsilon": m.c.eps})()
    for kernel in (None, "b200"):
        model = torch.nn.Module()
        model.attn = child
        assert A.patch_attention_blocks(model, kernel) == 1
        assert model.attn.attention_kernel == (kernel or "decomposed")
