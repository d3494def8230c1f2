"""What the 8-bit cache refuses, on the CPU: values that no answer is right for."""
import pytest
import torch

from shark_platform_b200 import _cabi as C
from shark_platform_b200 import attention as A


@pytest.mark.parametrize("softcap", [float("inf"), float("nan"), 0.0, -1.0, 1e39])
def test_softcaps_that_are_no_cap(softcap):
    cache = A.PagedKVCache(transformer_block_count=1, attn_head_count=2, attn_head_dim=64, dtype=torch.int8)
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(C.B200MoeError, match="softcap must be positive"):
        A.kv_attend(q, cache, cache.allocate(2), block_index=0, seq_block_ids=torch.zeros(1, 1, dtype=torch.int32),
                    seq_lens=torch.ones(1, dtype=torch.int32), softcap=softcap)


@pytest.mark.parametrize("softcap", [float("inf"), float("nan"), float("-inf")])
def test_the_c_abi_refuses_them_too(softcap):
    import ctypes

    desc, p = C.Kv8CacheDesc(2, 32, 8, 128, 16, 16, C.KV8_INT8), ctypes.c_void_p(4096)
    rc = C.lib.b200moe_kv8_attend(p, C.DT_BF16, 4096, p, p, ctypes.byref(desc), 0, p, p, 0, 1, 3, 32, 96, 0.1, softcap, p,
                                  C.DT_BF16, p, 1 << 30, None)
    assert rc == -1 and "softcap" in C.last_error()
