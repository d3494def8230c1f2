"""Attention over the 8- and 4-bit caches with softcaps far above the scores, up to the largest number."""
import pytest
import torch

import test_gpu_kv4 as four
import test_gpu_kv8 as eight
from oracle import kv4_oracle as k4

pytestmark = pytest.mark.gpu

BF, HF, F32 = four.BF, four.HF, four.F32


@pytest.mark.parametrize("io", [BF, HF, F32])
@pytest.mark.parametrize("softcap", [1e12, 1e30, 2e38, 3.4e38])
def test_four_bit(io, softcap):
    gen = torch.Generator().manual_seed(2)
    cache = four._cache(2, 64, 16)
    state, ids = k4.fill(cache, 22, gen), four._ids(1, 20, gen)
    four._attend_check(cache, state, ids, torch.tensor([290]), torch.randn(1, 2, 8, 64, generator=gen).to(io), softcap=softcap)


@pytest.mark.parametrize("code", [eight.I8, eight.E4])
@pytest.mark.parametrize("io", [BF, HF, F32])
@pytest.mark.parametrize("softcap", [1e30, 2e38, 3.4e38])
def test_eight_bit(code, io, softcap):
    eight._attend_case(code, io, 128, 8, 2, 32, 16, [90, 300], softcap=softcap)
