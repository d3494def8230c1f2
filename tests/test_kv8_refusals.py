"""What the 8-bit cache refuses, on the CPU: nothing here reaches a kernel."""
import ctypes

import pytest
import torch

from shark_platform_b200 import _cabi as C
from shark_platform_b200 import attention as A

DUMMY, OUT = ctypes.c_void_p(4096), ctypes.c_void_p(8192)


def _desc(**kw):
    d = dict(blocks=2, stride=32, kv_heads=8, head_dim=128, page_count=16, scale_block=16, code=C.KV8_INT8)
    d.update(kw)
    return C.Kv8CacheDesc(*(d[n] for n, _ in C.Kv8CacheDesc._fields_))


def _write(desc, q=DUMMY, qs=4096, ks=1024, vs=1024, io=C.DT_BF16, layer=1, order=0, bs=2, sl=4, pages=3, heads=32,
           scales=DUMMY, k=DUMMY, k_out=None):
    return C.lib.b200moe_attn_norm_rope_kv8_write(
        q, k, DUMMY, io, qs, ks, vs, None, None, 1e-5, OUT, k_out, DUMMY, scales, ctypes.byref(desc), layer, DUMMY,
        None, DUMMY, DUMMY, order, bs, sl, pages, heads, None)


def _attend(desc, q=DUMMY, qs=4096, new=1, bs=2, heads=32, scratch=DUMMY, nbytes=1 << 30, max_len=96, dt=C.DT_BF16, layer=0):
    return C.lib.b200moe_kv8_attend(q, dt, qs, DUMMY, DUMMY, ctypes.byref(desc), layer, DUMMY, DUMMY, bs, new, 3, heads,
                                    max_len, 0.1, 0.0, DUMMY, C.DT_BF16, scratch, nbytes, None)


def _read(desc, k=DUMMY, dt=C.DT_BF16, n=96, layer=0):
    return C.lib.b200moe_kv8_read(DUMMY, DUMMY, ctypes.byref(desc), layer, DUMMY, DUMMY, 2, 3, n, k, DUMMY, dt, None)


@pytest.mark.parametrize("bad", [dict(head_dim=96), dict(head_dim=256), dict(scale_block=0), dict(scale_block=3),
                                 dict(scale_block=128, stride=128), dict(scale_block=32, stride=48), dict(code=2),
                                 dict(stride=0), dict(kv_heads=0), dict(page_count=0), dict(blocks=0)])
def test_bad_geometry(bad):
    for call in (_write, _attend, _read):
        assert call(_desc(**bad)) == -1 and C.last_error()


def test_block_index_out_of_range():
    for call in (_write, _attend, _read):
        assert call(_desc(), layer=2) == -1 and call(_desc(), layer=-1) == -1


@pytest.mark.parametrize("kw,message", [
    (dict(heads=30), "multiple of the kv heads"), (dict(io=7), "dtype"), (dict(order=2), "rotation order"),
    (dict(q=ctypes.c_void_p(4104)), "16 bytes"), (dict(qs=4100), "16 bytes"), (dict(qs=2048), "shorter than the row"),
    (dict(ks=512), "shorter than the row"), (dict(q=None), "NULL"), (dict(scales=None), "scales"), (dict(sl=0), "sizes"),
    (dict(scales=ctypes.c_void_p(4100)), "scales"), (dict(bs=1 << 30, sl=4096), "too many"),
    (dict(k_out=DUMMY), "k_out")])
def test_write_refuses(kw, message):
    assert _write(_desc(), **kw) == -1 and message in C.last_error()


def test_plain_write_refuses():
    desc = C.KvCacheDesc(2, 32, 8, 128, 16)
    call = lambda d, dt: C.lib.b200moe_attn_norm_rope_kv_write(
        DUMMY, DUMMY, DUMMY, C.DT_BF16, 4096, 1024, 1024, None, None, 1e-5, OUT, None, DUMMY, dt, d, 0, DUMMY, None,
        DUMMY, DUMMY, 0, 2, 4, 3, 32, None)
    assert call(None, C.DT_BF16) == -1 and "NULL" in C.last_error()
    assert call(ctypes.byref(desc), 5) == -1 and "dtype" in C.last_error()
    desc.head_dim = 80
    assert call(ctypes.byref(desc), C.DT_BF16) == -1 and "head_dim" in C.last_error()


@pytest.mark.parametrize("kw,message", [
    (dict(new=0), "new_tokens"), (dict(new=17), "new_tokens"), (dict(heads=12), "multiple of the kv heads"),
    (dict(q=ctypes.c_void_p(4104)), "16 bytes"), (dict(qs=1024), "16 bytes"), (dict(scratch=None), "NULL"),
    (dict(scratch=ctypes.c_void_p(4104)), "16 bytes"), (dict(dt=9), "dtype"), (dict(bs=70000), "sizes"),
    (dict(max_len=0), "sizes")])
def test_attend_refuses(kw, message):
    assert _attend(_desc(), **kw) == -1 and message in C.last_error()


def test_attend_asks_for_its_scratch():
    d = _desc()
    need = C.lib.b200moe_kv8_attend_scratch_bytes(ctypes.byref(d), 2, 1, 32, 96)
    assert need > 0
    assert _attend(d, nbytes=need - 1) == -3 and "scratch" in C.last_error()
    assert C.lib.b200moe_kv8_attend_scratch_bytes(None, 2, 1, 32, 96) == 0
    assert C.lib.b200moe_kv8_attend_scratch_bytes(ctypes.byref(d), 0, 1, 32, 96) == 0


@pytest.mark.parametrize("kw,message", [(dict(k=ctypes.c_void_p(4100)), "16-byte"), (dict(dt=4), "dtype"),
                                        (dict(n=-1), "sizes"), (dict(k=None), "NULL")])
def test_read_refuses(kw, message):
    assert _read(_desc(), **kw) == -1 and message in C.last_error()


def test_empty_calls_do_nothing():
    assert _write(_desc(), bs=0) == 0 and _attend(_desc(), bs=0) == 0 and _read(_desc(), n=0) == 0


def _cache(dtype=torch.int8, stride=32, **kw):
    return A.PagedKVCache(transformer_block_count=2, attn_head_count=2, attn_head_dim=64, block_seq_stride=stride,
                          dtype=dtype, **kw)


def test_cache_geometry():
    c = _cache()
    slab, scales = c.allocate(5)
    assert c.quantized and c.scale_block == 16
    assert slab.dtype == torch.int8 and slab.shape == (5, 2 * 2 * 2 * 32 * 64)
    assert scales.dtype == torch.float32 and scales.shape == (5, 2 * 2 * 2 * 2)
    assert _cache(stride=20).scale_block == 4 and _cache(stride=7).scale_block == 1
    assert _cache(scale_block=32).scale_block == 32
    assert len(_cache(dtype=torch.bfloat16).allocate(2)) == 1
    for bad in (3, 0, 64, 128, -1):
        with pytest.raises(C.B200MoeError, match="scale_block"):
            _cache(scale_block=bad)
    with pytest.raises(C.B200MoeError, match="scale_block"):
        _cache(dtype=torch.float16, scale_block=16)


def _args(cache, bs=2, sl=3, heads=4, hd=64):
    q = torch.zeros(bs, sl, heads, hd, dtype=torch.bfloat16)
    k = torch.zeros(bs, sl, 2, hd, dtype=torch.bfloat16)
    kw = dict(block_index=1, seq_block_ids=torch.zeros(bs, 3, dtype=torch.int32),
              start_positions=torch.zeros(bs, dtype=torch.int32), freqs=torch.ones(hd // 2))
    return [q, k, k.clone(), cache, cache.allocate(4)], kw


@pytest.mark.parametrize("change,message", [
    (lambda a, k: a.__setitem__(0, a[0].half()), "alike"),
    (lambda a, k: a.__setitem__(0, a[0].double()), "fp32, fp16 or bf16"),
    (lambda a, k: a.__setitem__(0, a[0][:, :, :3]), "do not fit"),
    (lambda a, k: a.__setitem__(1, a[1][:, :2]), "do not fit"),
    (lambda a, k: a.__setitem__(4, a[4][:1]), "scales"),
    (lambda a, k: a[4].__setitem__(0, a[4][0].view(torch.float8_e4m3fn)), "must be"),
    (lambda a, k: a[4].__setitem__(0, a[4][0][:, :-8]), "page slab"),
    (lambda a, k: a[4].__setitem__(1, a[4][1][:2]), "scales"),
    (lambda a, k: k.update(block_index=2), "block_index"),
    (lambda a, k: k.update(seq_block_ids=k["seq_block_ids"][:1]), "seq_block_ids"),
    (lambda a, k: k.update(start_positions=k["start_positions"][:1]), "start_positions"),
    (lambda a, k: k.update(new_lens=torch.zeros(3)), "new_lens"),
    (lambda a, k: k.update(freqs=k["freqs"].double()), "freqs"),
    (lambda a, k: k.update(q_norm=torch.ones(32)), "norm weights"),
    (lambda a, k: k.update(k_norm=torch.ones(64).half()), "norm weights"),
    (lambda a, k: None, "CUDA tensor")])
def test_python_write_refuses(change, message):
    a, kw = _args(_cache())
    change(a, kw)
    with pytest.raises(C.B200MoeError, match=message):
        A.norm_rope_kv_write(*a, **kw)


def test_python_read_and_attend_refuse():
    cache = _cache()
    (q, _, _, _, state), kw = _args(cache)
    lens = torch.ones(2, dtype=torch.int32)
    base = dict(block_index=0, seq_block_ids=kw["seq_block_ids"])
    plain = _cache(dtype=torch.bfloat16)
    cases = [(lambda: A.kv_attend(q, plain, plain.allocate(4), seq_lens=lens, **base), "8-bit"),
             (lambda: A.kv_attend(q[:, :0], cache, state, seq_lens=lens, **base), "new tokens"),
             (lambda: A.kv_attend(q.repeat(1, 6, 1, 1), cache, state, seq_lens=lens, **base), "new tokens"),
             (lambda: A.kv_attend(q[..., :32], cache, state, seq_lens=lens, **base), "does not fit"),
             (lambda: A.kv_attend(q, cache, state, seq_lens=lens[:1], **base), "seq_lens"),
             (lambda: A.kv_attend(q, cache, state, seq_lens=lens, softcap=-1.0, **base), "softcap"),
             (lambda: A.kv_attend(q, cache, state, seq_lens=lens, out_dtype=torch.int8, **base), "fp32, fp16"),
             (lambda: A.kv_attend(q, cache, state, seq_lens=lens, **base), "CUDA tensor"),
             (lambda: A.kv_read(plain, plain.allocate(4), seq_lens=lens, **base), "8-bit"),
             (lambda: A.kv_read(cache, state, seq_lens=lens, dtype=torch.float64, **base), "fp32, fp16"),
             (lambda: A.kv_read(cache, state, seq_lens=lens[:1], **base), "seq_lens"),
             (lambda: A.kv_read(cache, state, seq_lens=lens, **base), "CUDA tensor")]
    for call, message in cases:
        with pytest.raises(C.B200MoeError, match=message):
            call()
