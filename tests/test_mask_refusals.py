"""What the look at masks refuses, on the CPU: nothing here reaches a kernel."""
import ctypes

import pytest

from shark_platform_b200 import _cabi as C

DUMMY = ctypes.c_void_p(4096)


def _check(mask=DUMMY, dt=C.DT_BF16, batch=64, row=8, masks=2, rows=8, columns=8, lens=None, bs=2, per=0):
    return C.lib.b200moe_causal_mask_check(mask, dt, batch, row, masks, rows, columns, lens, bs, per, None)


@pytest.mark.parametrize("kw,message", [
    (dict(mask=None), "NULL"), (dict(mask=ctypes.c_void_p(4097)), "aligned"), (dict(dt=5), "dtype"), (dict(columns=7), "sizes"),
    (dict(rows=-1), "sizes"), (dict(masks=-1), "sizes"), (dict(batch=-1), "sizes"), (dict(row=-8), "sizes"), (dict(bs=-1), "sizes"),
    (dict(per=-1), "sizes"), (dict(lens=DUMMY, per=2), "masks for"), (dict(lens=DUMMY, bs=3, per=1), "masks for")])
def test_refusals(kw, message):
    assert _check(**kw) == -1 and message in C.last_error()


def test_calls_without_work():
    assert _check(masks=0, bs=0) == 0 and _check(rows=0) == 0
