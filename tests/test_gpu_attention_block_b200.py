"""attention_kernel="b200" in the attention block: gradients."""
import pytest
import torch

from test_gpu_kv4_block import Model4
from test_gpu_kv8_block import I8, Model

pytestmark = pytest.mark.gpu


def _model(dtype, act=torch.float32, **kw):
    m = (Model4 if dtype == torch.uint8 else Model)(dtype, act=act, **kw)
    m.block.attention_kernel = "b200"
    return m


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
