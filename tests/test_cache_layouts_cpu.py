"""Layouts of caches and weights that the calls take, and those that they refuse, by address alone (no GPU)."""

import itertools
import random

import pytest
import torch

import flash_topk_attn_v2 as fta
from flash_topk_attn_v2 import _lib, cache_evict, q4_cache

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
    _, _, nbytes, _, _ = cache_evict._moved_layout("evict", True, cache_evict._metas((*c, w)), 1, 1, 10, True)
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
        _, _, nbytes, _, _ = cache_evict._moved_layout("evict", True, cache_evict._metas((*bad, w)), 1, 1, 2, True)
        with pytest.raises(ValueError, match="aligned"):
            cache_evict._check_aligned("evict", True, nbytes, [t.data_ptr() for t in (*bad, w)])


def _bytes(shape, stride, size, at):
    """Every byte of a tensor."""
    found = set()
    for i in itertools.product(*map(range, shape)):
        a = at + size * sum(x * s for x, s in zip(i, stride))
        found.update(range(a, a + size))
    return found


def test_tensors_that_share_a_byte():
    """Any strides, runs between each other, types of different sizes: against the sets of their bytes."""
    rng = random.Random(1)
    seen = {False: 0, True: 0}
    for _ in range(4000):
        a, b = ((tuple(rng.randint(1, 5) for _ in range(d)), tuple(rng.choice([0, 1, 2, 3, 4, 5, 7, 8, 12, 16, 20, 40]) for _ in range(d)),
                 rng.choice([1, 2, 4])) for d in (rng.randint(1, 3), rng.randint(1, 3)))
        delta = rng.randint(-150, 150)
        meet = bool(_bytes(*a, 0) & _bytes(*b, delta))
        seen[meet] += 1
        assert _lib.tensors_meet(a, b, delta) == meet, (a, b, delta)
    assert min(seen.values()) > 500


def test_weights_lie_apart_from_what_is_read():
    B, Hk, S, C = 3, 2, 16, 64
    raw = torch.zeros(B, 2 * S * C + 2 * Hk * S + 8, dtype=torch.bfloat16)  # a request's keys, values and weights side by side
    keys = raw[:, :S * C].view(B, S, C)
    w = raw[:, 2 * S * C:2 * S * C + 2 * Hk * S].view(torch.float32).view(B, Hk, S)
    apart = lambda *t: _lib.check_apart("weights", "weights", w, *t)  # noqa: E731
    apart(keys, raw[:, S * C:2 * S * C].view(B, S, C), torch.zeros(B, 4, 1), raw[0, -8:].view(torch.int32)[:B])
    for bad in (w, w[1:2, 1:], keys[:, :, :1].as_strided((B, S, C), keys.stride(), S * C + 64), raw, raw.view(torch.int32)[2, S * C + 2:][:B]):
        with pytest.raises(ValueError, match="overlap"):
            apart(bad)


def _arena(B, Hk, S, D):
    """One buffer a request: its key and value codes, their scales and its weights side by side."""
    G = -(-D // 32)
    sizes = [16 * G * Hk * S, -(-2 * G * Hk * S // 16) * 16] * 2 + [4 * Hk * S]
    raw = torch.zeros(B, -(-sum(sizes) // 16) * 16, dtype=torch.uint8)
    parts, at = [], 0
    for n in sizes:
        parts.append(raw[:, at:at + n])
        at += n
    codes = [parts[i].view(B, Hk, S, 16 * G) for i in (0, 2)]
    scales = [parts[i][:, :2 * G * Hk * S].view(torch.float16).view(B, Hk, S, G) for i in (1, 3)]
    return fta.Q4Cache(codes[0], scales[0], codes[1], scales[1]), parts[4].view(torch.float32).view(B, Hk, S)


@pytest.mark.parametrize("D", [48, 64, 96])
def test_requests_that_lie_between_each_other(D):
    """No two rows share memory, whatever the tensors' spans."""
    B, Hk, S = 3, 2, 16
    c, w = _arena(B, Hk, S, D)
    q4_cache.check_q4_written("cache", c)
    metas, at = cache_evict._metas((*c, w)), [t.data_ptr() for t in (*c, w)]
    cache_evict._check_apart("evict", True, metas, metas, at, at, True)
    # and half of the requests into the other half's places
    c2, w2 = _arena(2 * B, Hk, S, D)
    halves = [(fta.Q4Cache(*(t[i::2] for t in c2)), w2[i::2]) for i in (0, 1)]
    m, a = zip(*((cache_evict._metas((*x, y)), [t.data_ptr() for t in (*x, y)]) for x, y in halves))
    cache_evict._check_apart("evict", True, m[0], m[1], a[0], a[1])
    pool = torch.zeros(B, 2, 2, S, Hk * D, dtype=torch.bfloat16)
    kv = [(cache_evict._metas((pool[:, i, 0], pool[:, i, 1], w)), [pool[:, i, j].data_ptr() for j in (0, 1)] + [1 << 40]) for i in (0, 1)]
    kv[1][1][2] = 1 << 41
    cache_evict._check_apart("evict", False, kv[0][0], kv[1][0], kv[0][1], kv[1][1])
    # a byte too many
    a = list(at)
    for i, j in ((0, 1), (1, 2), (2, 3), (3, 4)):
        b = list(at)
        b[j] -= 16 if j % 2 == 0 else 4
        with pytest.raises(ValueError, match="share memory|overlap"):
            cache_evict._check_apart("evict", True, metas, metas, b, b, True)
    a[4] += 4 * Hk * S  # the weights of one request in the next one's codes
    with pytest.raises(ValueError, match="weights overlap"):
        cache_evict._check_apart("evict", True, metas, metas, a, a, True)


def test_weights_that_are_read_may_be_shared():
    """By heads, for instance, of an eviction into another cache; where they are written they may not."""
    c, w = fta.flash_q4_cache(3, 16, 2, 64, "cpu"), torch.zeros(3, 1, 16).expand(3, 2, 16)
    layout = cache_evict._moved_layout("evict", True, cache_evict._metas((*c, w)), 3, 2, 5, False)
    assert list(layout[3]) == [16, 0]
    with pytest.raises(ValueError, match="share memory"):
        cache_evict._moved_layout("evict", True, cache_evict._metas((*c, w)), 3, 2, 5, True)
