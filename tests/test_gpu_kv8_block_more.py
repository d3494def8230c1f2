"""Calls of B200PagedAttentionBlock that its caches have no answer for."""
import pytest
import torch

from test_gpu_kv8_block import E4, I8, Model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norms,use_hf,padded", [(True, False, False), (False, True, False), (False, False, True)])
def test_a_continued_prompt_over_a_plain_cache(norms, use_hf, padded):
    """The one-pass write takes it, but nothing would attend the cached positions."""
    from shark_platform_b200 import _cabi as C

    m = Model(torch.float32, norms, use_hf)
    kw = dict(new_lens=torch.tensor([16, 9]).cuda()) if padded else {}
    m.call(m.rows(16), start_index=0, **kw)
    before = m.state[0].clone()
    for start in (16, -1):
        with pytest.raises(C.B200MoeError, match="continued prompts"):
            m.call(m.rows(16), start_index=start, **kw)
    assert torch.equal(m.state[0], before)
    plain = Model(torch.float32)  # as before: the new positions only, as the reference does
    assert torch.isfinite(plain.call(plain.rows(16), start_index=16)).all()


@pytest.mark.parametrize("dtype", [I8, E4])
def test_a_prompt_before_the_first_position(dtype):
    from shark_platform_b200 import _cabi as C

    m = Model(dtype)
    with pytest.raises(C.B200MoeError, match="continued prompts"):
        m.call(m.rows(16), start_index=-1)
    assert not m.state[0].view(torch.uint8).any()
