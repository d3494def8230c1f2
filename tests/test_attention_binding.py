"""The compiled torch binding of the cache operators: who loads it, and what happens where it
does not load."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_the_package_imports_without_it():
    """The MoE layers, linears, loader, plugin and the attention block's module load the C library only."""
    _run("""
import shark_platform_b200._cabi as C
C.OPS_PATH = "/nonexistent/_attention_ops.so"
from shark_platform_b200 import attention, gguf_io, moe, ops, parallel, plugin, types
assert "_attention_ops" not in open("/proc/self/maps").read()
attention.PagedKVCache(transformer_block_count=1, attn_head_count=1, attn_head_dim=64).allocate(1)
""")


def test_the_first_cache_operator_loads_it():
    _run("""
import torch
from shark_platform_b200 import _cabi as C, attention as A
cache = A.PagedKVCache(transformer_block_count=1, attn_head_count=1, attn_head_dim=64, dtype=torch.int8)
try:
    A.kv_read(cache, cache.allocate(1), block_index=0, seq_block_ids=torch.zeros(1, 1, dtype=torch.int32),
              seq_lens=torch.zeros(1, dtype=torch.int32))
except C.B200MoeError as e:
    assert "CUDA tensor" in str(e), e
assert "_attention_ops.so" in open("/proc/self/maps").read()
assert C.attention_ops is C.attention_ops and not hasattr(C, "attention_opz")
""")


@pytest.mark.parametrize("what", ["missing", "not a library"])
def test_a_binding_that_does_not_load(what, monkeypatch, tmp_path):
    from shark_platform_b200 import _cabi as C, attention as A

    path = tmp_path / "_attention_ops.so"
    if what != "missing":
        path.write_text("no library")
    monkeypatch.delitem(C.__dict__, "attention_ops", raising=False)
    monkeypatch.setattr(C, "OPS_PATH", str(path))
    cache = A.PagedKVCache(transformer_block_count=1, attn_head_count=1, attn_head_dim=64, dtype=torch.int8)
    with pytest.raises(C.B200MoeError, match="shark_platform_b200.build"):
        A.kv_read(cache, cache.allocate(1), block_index=0, seq_block_ids=torch.zeros(1, 1, dtype=torch.int32),
                  seq_lens=torch.zeros(1, dtype=torch.int32))
    assert "attention_ops" not in C.__dict__
