"""Layouts of caches and weights that the calls take, and those that they refuse, by address alone (no GPU)."""

import pytest
import torch

import flash_topk_attn_v2 as fta
from flash_topk_attn_v2 import cache_evict, q4_cache

CPU = torch.device("cpu")


def _request(D, S=75):
    """The second request of a contiguous cache of two, one head: its scales start 75 rows in."""
    return fta.Q4Cache(*(t[1:] for t in fta.flash_q4_cache(2, S, 1, D, "cpu")))


@pytest.mark.parametrize("D", [16, 32, 80, 96, 144, 160, 208, 224])
def test_scales_of_an_odd_number_of_groups_start_anywhere(D):
    c = _request(D)
    S, args = q4_cache.q4_args("cache", c, 1, 1, D, CPU, write=True)
    assert S == 75 and args[2] == c.k_scales.data_ptr() and args[2] % 4 == 2
    at = [t.data_ptr() for t in c] + [64]
    w = torch.zeros(1, 1, 75)
    _, _, nbytes, _, _ = cache_evict._moved_layout("evict", True, cache_evict._metas((*c, w)), 1, 1, 10)
    cache_evict._check_aligned("evict", True, nbytes, at)


@pytest.mark.parametrize("D", [48, 64, 128, 192, 256])
def test_scales_that_are_read_by_pairs_start_at_pairs(D):
    """Where D fills an even number of groups, and codes always at 16 bytes."""
    S, G = 4, -(-D // 32)
    c = fta.flash_q4_cache(1, S, 1, D, "cpu")
    q4_cache.q4_args("cache", c, 1, 1, D, CPU)
    raw = torch.zeros(S * G + 2, dtype=torch.float16)
    scales = raw[1 + raw.data_ptr() // 2 % 2:][:S * G].view(1, 1, S, G)
    codes = torch.zeros(16 * G * S + 32, dtype=torch.uint8)
    codes = codes[(-codes.data_ptr()) % 16 + 8:][:16 * G * S].view(1, 1, S, 16 * G)
    assert scales.data_ptr() % 4 == 2
    w = torch.zeros(1, 1, S)
    for bad in (c._replace(k_scales=scales), c._replace(v_scales=scales), c._replace(k_codes=codes), c._replace(v_codes=codes)):
        with pytest.raises(ValueError, match="aligned"):
            q4_cache.q4_args("cache", bad, 1, 1, D, CPU)
        _, _, nbytes, _, _ = cache_evict._moved_layout("evict", True, cache_evict._metas((*bad, w)), 1, 1, 2)
        with pytest.raises(ValueError, match="aligned"):
            cache_evict._check_aligned("evict", True, nbytes, [t.data_ptr() for t in (*bad, w)])
