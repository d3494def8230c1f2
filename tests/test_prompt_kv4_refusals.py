"""What prompt_attend and the 4-bit cache refuse, on the CPU: nothing here reaches a kernel."""
import ctypes
import math

import pytest
import torch

from shark_platform_b200 import _cabi as C
from shark_platform_b200 import attention as A

DUMMY, OUT, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(8192), ctypes.c_void_p(4104)


def _desc(**kw):
    d = dict(blocks=2, stride=32, kv_heads=8, head_dim=128, page_count=16)
    d.update(kw)
    return C.KvCacheDesc(*(d[n] for n, _ in C.KvCacheDesc._fields_))


def _write(desc, q=DUMMY, qs=4096, ks=1024, vs=1024, io=C.DT_BF16, layer=1, order=0, bs=2, sl=4, pages=3, heads=32,
           scales=DUMMY, k=DUMMY, k_out=None):
    return C.lib.b200moe_attn_norm_rope_kv4_write(
        q, k, DUMMY, io, qs, ks, vs, None, None, 1e-5, OUT, k_out, DUMMY, scales, ctypes.byref(desc), layer, DUMMY,
        None, DUMMY, DUMMY, order, bs, sl, pages, heads, None)


def _attend(desc, q=DUMMY, qs=4096, new=1, bs=2, heads=32, scratch=DUMMY, nbytes=1 << 30, max_len=96, dt=C.DT_BF16, layer=0,
            softcap=0.0, pages=3, scales=DUMMY):
    return C.lib.b200moe_kv4_attend(q, dt, qs, DUMMY, scales, ctypes.byref(desc), layer, DUMMY, DUMMY, bs, new, pages, heads,
                                    max_len, 0.1, softcap, DUMMY, C.DT_BF16, scratch, nbytes, None)


def _read(desc, k=DUMMY, dt=C.DT_BF16, n=96, layer=0, scales=DUMMY, bs=2):
    return C.lib.b200moe_kv4_read(DUMMY, scales, ctypes.byref(desc), layer, DUMMY, DUMMY, bs, 3, n, k, DUMMY, dt, None)


@pytest.mark.parametrize("bad", [dict(head_dim=96), dict(head_dim=256), dict(stride=0), dict(kv_heads=0), dict(page_count=0),
                                 dict(blocks=0), dict(kv_heads=70000), dict(page_count=1 << 30)])
def test_bad_geometry(bad):
    for call in (_write, _attend, _read):
        assert call(_desc(**bad)) == -1 and C.last_error()


def test_block_index_out_of_range():
    for call in (_write, _attend, _read):
        assert call(_desc(), layer=2) == -1 and call(_desc(), layer=-1) == -1


@pytest.mark.parametrize("kw,message", [
    (dict(heads=30), "multiple of the kv heads"), (dict(io=7), "dtype"), (dict(order=2), "rotation order"),
    (dict(q=ODD), "16 bytes"), (dict(qs=4100), "16 bytes"), (dict(qs=2048), "shorter than the row"),
    (dict(ks=512), "shorter than the row"), (dict(q=None), "NULL"), (dict(scales=None), "scales"), (dict(sl=0), "sizes"),
    (dict(scales=ODD), "scales"), (dict(bs=1 << 30, sl=4096), "too many"), (dict(k_out=DUMMY), "k_out")])
def test_write_refuses(kw, message):
    assert _write(_desc(), **kw) == -1 and message in C.last_error()


@pytest.mark.parametrize("kw,message", [
    (dict(new=0), "new_tokens"), (dict(new=17), "new_tokens"), (dict(heads=12), "multiple of the kv heads"),
    (dict(q=ODD), "16 bytes"), (dict(qs=1024), "16 bytes"), (dict(scratch=None), "NULL"), (dict(scratch=ODD), "16 bytes"),
    (dict(dt=9), "dtype"), (dict(bs=70000), "sizes"), (dict(max_len=0), "sizes"), (dict(softcap=math.inf), "softcap"),
    (dict(softcap=math.nan), "softcap"), (dict(pages=1 << 26), "positions"), (dict(scales=ODD), "16 bytes")])
def test_attend_refuses(kw, message):
    assert _attend(_desc(), **kw) == -1 and message in C.last_error()


@pytest.mark.parametrize("kw,message", [(dict(k=None), "NULL"), (dict(k=ODD), "16-byte"), (dict(dt=4), "dtype"), (dict(n=-1), "sizes"),
                                        (dict(bs=70000), "sizes"), (dict(scales=ODD), "16-byte")])
def test_read_refuses(kw, message):
    assert _read(_desc(), **kw) == -1 and message in C.last_error()


def test_attend_asks_for_its_scratch():
    d = _desc()
    need = C.lib.b200moe_kv4_attend_scratch_bytes(ctypes.byref(d), 2, 1, 32, 96)
    assert need > 0 and _attend(d, nbytes=need - 1) == -3 and "scratch" in C.last_error()
    assert C.lib.b200moe_kv4_attend_scratch_bytes(ctypes.byref(d), 2, 17, 32, 96) == 0
    assert C.lib.b200moe_kv4_attend_scratch_bytes(None, 2, 1, 32, 96) == 0


def test_calls_without_work():
    assert _write(_desc(), bs=0) == 0 and _attend(_desc(), bs=0) == 0 and _read(_desc(), bs=0) == 0 and _read(_desc(), n=0) == 0


# ------------------------------------------------------------------------ prompts
def _prompt(q=DUMMY, k=DUMMY, v=DUMMY, dt=C.DT_BF16, qs=4096, ks=1024, vs=1024, cu=DUMMY, bs=2, rows=10, krows=10, heads=32, kvh=8,
            hd=128, softcap=0.0, out=OUT, odt=C.DT_BF16, scratch=DUMMY, nbytes=1 << 40):
    return C.lib.b200moe_prompt_attend(q, k, v, dt, qs, ks, vs, cu, None, bs, rows, krows, heads, kvh, hd, 0.1, softcap, out, odt, scratch,
                                       nbytes, None)


@pytest.mark.parametrize("kw,message", [
    (dict(heads=30), "multiple of the kv heads"), (dict(dt=3), "dtype"), (dict(odt=9), "dtype"), (dict(hd=80), "head_dim"),
    (dict(q=ODD), "16 bytes"), (dict(qs=4100), "16 bytes"), (dict(vs=1028), "16 bytes"), (dict(qs=2048), "shorter than the row"),
    (dict(ks=512), "shorter than the row"), (dict(q=None), "NULL"), (dict(v=None), "NULL"), (dict(cu=None), "NULL"),
    (dict(out=None), "NULL"), (dict(out=ctypes.c_void_p(8208)), "32-byte"), (dict(bs=-1), "sizes"), (dict(rows=-1), "sizes"), (dict(rows=1 << 31), "2^31"),
    (dict(softcap=math.inf), "softcap"), (dict(heads=1 << 20, qs=1 << 27), "heads")])
def test_prompt_refuses(kw, message):
    assert _prompt(**kw) == -1 and message in C.last_error()


def test_prompt_asks_for_its_scratch():
    """Few rows and long keys: the keys are split, and the parts need room."""
    size = lambda *a: C.lib.b200moe_prompt_attend_scratch_bytes(*a)
    need = size(C.DT_BF16, 1, 8, 20000, 32, 8, 128)
    assert need > 0 and need % (8 * 32 * 132 * 4) == 0
    kw = dict(bs=1, rows=8, krows=20000)
    assert _prompt(**kw, nbytes=need - 1) == -3 and "scratch" in C.last_error()
    assert _prompt(**kw, scratch=None) == -1 and "scratch" in C.last_error()
    assert _prompt(**kw, scratch=ODD) == -1 and "scratch" in C.last_error()
    assert size(C.DT_BF16, 1, 16384, 16384, 32, 8, 128) == 0 and size(C.DT_F32, 1, 8, 20000, 32, 8, 128) == 0
    assert size(C.DT_BF16, 0, 8, 20000, 32, 8, 128) == 0 and size(C.DT_BF16, 1, 8, 0, 32, 8, 128) == 0


def test_prompt_without_rows():
    assert _prompt(rows=0) == 0


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("change,message", [
    (dict(q=_t(10, 4, 96), k=_t(10, 2, 96), v=_t(10, 2, 96)), "head_dim 64 or 128"), (dict(q=_t(10, 3, 64)), "multiple"),
    (dict(q=_t(1, 10, 4, 64)), "must be"), (dict(v=_t(9, 2, 64)), "must be"), (dict(k=_t(10, 2, 64, dtype=torch.float32)), "alike"),
    (dict(q=_t(10, 4, 64, dtype=torch.int8)), "alike"), (dict(cu_seqlens=torch.zeros(2, 2, dtype=torch.int32)), "whole number"),
    (dict(cu_seqlens=torch.zeros(3)), "whole number"), (dict(cu_seqlens=torch.zeros(0, dtype=torch.int32)), "whole number"),
    (dict(cu_seqlens_k=torch.zeros(4, dtype=torch.int32)), "other sequences"),
    (dict(k=_t(12, 2, 64), v=_t(12, 2, 64)), "cu_seqlens_k says"), (dict(softcap=0.0), "softcap"), (dict(softcap=-1.0), "softcap"),
    (dict(softcap=math.inf), "softcap"), (dict(out_dtype=torch.int8), "alike"), (dict(q=_t(10, 4, 64).requires_grad_()), "no gradient"),
    (dict(v=_t(10, 2, 64).requires_grad_()), "no gradient"), (dict(), "CUDA tensor"), (dict(k=3), "tensor")])
def test_prompt_attend_refuses(change, message):
    kw = dict(q=_t(10, 4, 64), k=_t(10, 2, 64), v=_t(10, 2, 64), cu_seqlens=torch.tensor([0, 4, 10]))
    kw.update(change)
    with pytest.raises(C.B200MoeError, match=message):
        A.prompt_attend(kw.pop("q"), kw.pop("k"), kw.pop("v"), **kw)


def test_prompt_attend_without_gradients_may_have_inputs_that_want_them():
    with torch.no_grad(), pytest.raises(C.B200MoeError, match="CUDA tensor"):
        A.prompt_attend(_t(10, 4, 64).requires_grad_(), _t(10, 2, 64), _t(10, 2, 64), cu_seqlens=torch.tensor([0, 10]))


# -------------------------------------------------------------------- the cache's class
def test_four_bit_cache():
    c = A.PagedKVCache(transformer_block_count=3, attn_head_count=2, attn_head_dim=128, block_seq_stride=24, dtype=torch.uint8)
    slab, scales = c.allocate(5)
    assert c.quantized and slab.dtype == torch.uint8 and slab.shape == (5, 3 * 2 * 2 * 24 * 64)
    assert scales.dtype == torch.float16 and scales.shape == (5, 3 * 2 * 2 * 24 * 4 * 2)
    with pytest.raises(C.B200MoeError, match="scale_block"):
        A.PagedKVCache(transformer_block_count=1, attn_head_count=1, attn_head_dim=64, dtype=torch.uint8, scale_block=16)
    with pytest.raises(C.B200MoeError, match="head_dim"):
        A.PagedKVCache(transformer_block_count=1, attn_head_count=1, attn_head_dim=80, dtype=torch.uint8)


def _state_calls(cache, state):
    ids, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, k = _t(1, 1, 4, 64), _t(1, 1, 2, 64)
    return (lambda: A.kv_read(cache, state, block_index=0, seq_block_ids=ids, seq_lens=lens),
            lambda: A.kv_attend(q, cache, state, block_index=0, seq_block_ids=ids, seq_lens=lens),
            lambda: A.norm_rope_kv_write(q, k, k, cache, state, block_index=0, seq_block_ids=ids, start_positions=lens,
                                         freqs=torch.ones(32)))


def test_state_of_another_cache():
    make = lambda dt: A.PagedKVCache(transformer_block_count=1, attn_head_count=2, attn_head_dim=64, dtype=dt)
    four, eight, plain = make(torch.uint8), make(torch.int8), make(torch.bfloat16)
    state = four.allocate(2)
    wrong = [(four, eight.allocate(2), "page slab|fp16"), (eight, state, "page slab"), (four, plain.allocate(2), "page slab"),
             (four, state[:1], "scales"), (four, [state[0], state[1].float()], "fp16"), (four, [state[0], state[1][:, :4]], "fp16"),
             (four, [state[0], state[1][:1]], "fp16"), (four, [state[0].to(torch.int8), state[1]], "Byte"), (four, state, "CUDA tensor")]
    for cache, st, message in wrong:
        for call in _state_calls(cache, st):
            with pytest.raises(C.B200MoeError, match=message):
                call()
