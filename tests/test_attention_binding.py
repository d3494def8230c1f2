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


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """What build() would run, with nothing run; everything but the binding is up to date."""
    from shark_platform_b200 import build as B

    ops, stamp = tmp_path / "_attention_ops.so", tmp_path / "attention_ops.stamp"
    ops.write_bytes(b"")
    monkeypatch.setattr(B, "OPS", str(ops))
    stamp.write_text(B._ops_stamp())  # the command names the output
    monkeypatch.setattr(B, "OPS_STAMP", str(stamp))
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(B.subprocess, "run", run)

    def build():
        ran.clear()
        B.build()
        return [c for c in ran if any(str(a).endswith("attention_ops.cpp") for a in c)]

    return build, stamp, monkeypatch


def test_an_up_to_date_binding_is_kept(commands):
    build, stamp, _ = commands
    assert build() == []


@pytest.mark.parametrize("what", ["torch", "python", "flags", "no stamp", "library"])
def test_the_binding_is_built_again(commands, what):
    from shark_platform_b200 import build as B

    build, stamp, monkeypatch = commands
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9")
    elif what == "python":
        import sysconfig

        monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-399")
    elif what == "flags":
        monkeypatch.setattr(B, "CXX", "another-compiler")
    elif what == "no stamp":
        stamp.unlink()
    else:
        os.unlink(B.OPS)
    assert len(build()) == 1
    assert stamp.read_text() == B._ops_stamp()
    if what != "library":
        assert build() == []  # and not a second time


def test_the_c_library_is_built_without_torch(commands):
    import importlib.util

    build, stamp, monkeypatch = commands
    stamp.unlink()
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setitem(sys.modules, "torch", None)  # an import of it fails
    assert build() == []
    assert not stamp.exists()
