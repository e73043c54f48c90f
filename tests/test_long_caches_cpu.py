"""What of 4-bit caches, key weights and eviction is checked without a GPU: sizes, layouts, argument checks."""

import ctypes

import pytest
import torch

import flash_topk_attn_v2 as fta
from flash_topk_attn_v2 import _lib, cache_evict, q4_cache

X = 4096  # an address that nothing reads


def _s(*v):
    return _lib.i64arr(v)


def _attn(B=1, H=4, Hk=2, T=1, S=64, D=64, left=64, sinks=0, scale=0.1, dtype=0, kc=X, kcs=(0, 0), ks=X, kss=(0, 0), q=X, ws=None,
          nbytes=0):
    z3 = _s(0, 0, 0)
    return _lib.lib().fta_q4_attn(q, z3, kc, _s(*kcs), ks, _s(*kss), X, _s(0, 0), X, _s(0, 0), dtype, B, H, Hk, T, S, D, X, left,
                                  sinks, scale, X, z3, X, ws, nbytes, None)


@pytest.mark.parametrize("args", [dict(B=0), dict(H=3), dict(T=0), dict(S=0), dict(D=24), dict(D=272), dict(left=-1), dict(sinks=-1),
                                  dict(scale=0.0), dict(scale=3e38), dict(dtype=2), dict(kc=X + 8), dict(kcs=(8, 0)), dict(ks=X + 2),
                                  dict(kss=(1, 0)), dict(q=None), dict(S=100000, left=100000), dict(kc=None)], ids=str)
def test_attention_argument_errors(args):
    assert _attn(**args) == _lib.FTA_ERR_ARG and _lib.lib().fta_last_error()


@pytest.mark.parametrize("args", [dict(S=1 << 30), dict(T=1 << 21, H=1 << 10, Hk=1), dict(H=1 << 21, Hk=1), dict(B=1 << 30, Hk=1 << 20, H=1 << 20),
                                  dict(B=1 << 23, H=2, Hk=2)], ids=str)
def test_attention_limits(args):
    assert _attn(**args) == _lib.FTA_ERR_UNSUPPORTED
    a = dict(B=1, H=4, Hk=2, T=1, S=64, D=64, left=64, sinks=0) | args
    assert _lib.lib().fta_q4_attn_workspace_size(*(a[n] for n in ("B", "H", "Hk", "T", "S", "D", "left", "sinks"))) == 0


def _weigh(B=1, H=4, Hk=2, T=1, S=64, D=64, left=64, sinks=0, scale=0.1, dtype=0, q=X, k=X, ks=None, kss=None, nbytes=0):
    z3, z2 = _s(0, 0, 0), _s(0, 0)
    return _lib.lib().fta_cache_weights(q, z3, k, z3, ks, kss, dtype, B, H, Hk, T, S, D, X, left, sinks, scale, X, X, z2, None, nbytes,
                                        None)


@pytest.mark.parametrize("args", [dict(B=0), dict(H=3), dict(T=0), dict(S=0), dict(D=24), dict(D=272), dict(left=-1), dict(sinks=-1),
                                  dict(scale=0.0), dict(scale=3e38), dict(dtype=2), dict(q=None), dict(k=None), dict(ks=X),
                                  dict(k=X + 8, ks=X, kss=_s(0, 0)), dict(T=4096, S=4096, left=4096)], ids=lambda a: "-".join(a))
def test_weights_argument_errors(args):
    assert _weigh(**args) == _lib.FTA_ERR_ARG and _lib.lib().fta_last_error()


@pytest.mark.parametrize("args", [dict(S=1 << 30), dict(T=1 << 30), dict(B=1 << 17, T=100), dict(B=1 << 30, T=1 << 28, H=1 << 20, Hk=1),
                                  dict(S=1 << 29, T=1 << 29, B=100)], ids=str)
def test_weights_limits(args):
    assert _weigh(**args) == _lib.FTA_ERR_UNSUPPORTED


def _evict(tensors=2, B=1, Hk=1, S=64, S_out=64, budget=8, recent=0, sinks=0, rows=(128, 128, 128, 128), src=X, dst=X, w=X, wo=X, stride=128):
    n = max(tensors, 1)
    P = ctypes.c_void_p * n
    st = _s(*(stride,) * (3 * n))
    return _lib.lib().fta_cache_evict(tensors, P(*(src,) * n), st, P(*(dst,) * n), st, (ctypes.c_int32 * 4)(*rows), w, _s(0, 0), wo, _s(0, 0),
                                      B, Hk, S, S_out, budget, recent, sinks, X, X, X, None)


@pytest.mark.parametrize("args", [dict(B=0), dict(budget=0), dict(budget=65), dict(S_out=7), dict(tensors=0), dict(tensors=5),
                                  dict(recent=5, sinks=4), dict(recent=-1), dict(sinks=-1), dict(rows=(0, 128)), dict(rows=(128, 514)),
                                  dict(rows=(3, 128)), dict(dst=2 * X), dict(wo=2 * X), dict(src=None, dst=None), dict(w=None),
                                  dict(stride=129), dict(src=X + 1, dst=X + 1)], ids=str)
def test_eviction_argument_errors(args):
    assert _evict(**args) == _lib.FTA_ERR_ARG and _lib.lib().fta_last_error()


@pytest.mark.parametrize("args", [dict(S=1 << 30), dict(S_out=1 << 30), dict(B=1 << 22), dict(Hk=1 << 21), dict(B=1 << 30, S=1 << 28)], ids=str)
def test_eviction_limits(args):
    assert _evict(**args) == _lib.FTA_ERR_UNSUPPORTED


def test_read_and_append_argument_errors():
    L, z2, z3 = _lib.lib(), _s(0, 0), _s(0, 0, 0)
    read = lambda at=X, dt=0, D=64, S=8, st=z2: L.fta_q4_read(at, st, X, z2, X, z2, X, z2, dt, 1, 2, S, D, X, X, None)  # noqa: E731
    assert {read(at=X + 4), read(at=None), read(dt=2), read(D=20), read(S=0), read(st=_s(4, 0))} == {_lib.FTA_ERR_ARG}
    assert read(S=1 << 30) == _lib.FTA_ERR_UNSUPPORTED

    def append(k=X, D=64, S=8, eps=1e-6, R=64, codes=X, cs=z2):
        return L.fta_qk_norm_rope_append_q4(X, z3, k, z3, X, z3, 0, 1, 4, 2, 1, D, None, None, 2, X, X, 8, R, 0, None, eps, 0, X, S, X,
                                            z3, codes, cs, X, z2, X, z2, X, z2, None)

    assert {append(k=None), append(D=24), append(S=0), append(eps=0.0), append(R=80), append(codes=None), append(codes=X + 2),
            append(cs=_s(2, 0))} == {_lib.FTA_ERR_ARG}


def test_a_cache_and_its_layouts():
    B, S, Hk, D = 3, 5, 2, 80
    c = fta.flash_q4_cache(B, S, Hk, D, "cpu")
    assert [tuple(t.shape) for t in c] == [(B, Hk, S, 48), (B, Hk, S, 3)] * 2
    assert [t.dtype for t in c] == [torch.uint8, torch.float16] * 2 and all(int(t.count_nonzero()) == 0 for t in c)
    q4_cache.check_q4_written("cache", c)
    # one allocation for keys and values, side by side or in turn
    codes, scales = torch.zeros(B, 2, Hk, S, 48, dtype=torch.uint8), torch.zeros(2, B, Hk, S, 3, dtype=torch.float16)
    q4_cache.check_q4_written("cache", fta.Q4Cache(codes[:, 0], scales[0], codes[:, 1], scales[1]))
    codes = torch.zeros(B, Hk, 2, S, 48, dtype=torch.uint8)
    q4_cache.check_q4_written("cache", fta.Q4Cache(codes[:, :, 0], c.k_scales, codes[:, :, 1], c.v_scales))
    raw = torch.zeros(B * Hk * S * 48 + 6 * B * Hk * S, dtype=torch.uint8)
    overlap = raw[:B * Hk * S * 6].view(torch.float16).view(B, Hk, S, 3)
    for bad in (c._replace(v_codes=c.k_codes), c._replace(v_scales=c.k_scales), c._replace(k_codes=c.k_codes[:1].expand(B, -1, -1, -1)),
                c._replace(k_scales=c.k_scales[:, :1].expand(-1, Hk, -1, -1)),
                c._replace(k_codes=raw[:B * Hk * S * 48].view(B, Hk, S, 48), k_scales=overlap),
                c._replace(k_codes=raw[:B * Hk * S * 48].view(B, Hk, S, 48), v_codes=raw[16:16 + B * Hk * S * 48].view(B, Hk, S, 48))):
        with pytest.raises(ValueError, match="share memory"):
            q4_cache.check_q4_written("cache", bad)


def test_cpu_tensors_are_refused():
    q, c, ln = torch.zeros(1, 1, 64, dtype=torch.float16), fta.flash_q4_cache(1, 4, 1, 64, "cpu"), torch.zeros(1, dtype=torch.int32)
    t = torch.zeros(4, 32)
    for f in (lambda: fta.flash_window_attn_decode_q4(q, c, ln, 1, 4), lambda: fta.flash_q4_cache_read(c, 64, torch.float16),
              lambda: fta.flash_qk_norm_rope_append_q4(q, q, q, c, ln, 1, t, t),
              lambda: fta.flash_cache_weights(q, c, torch.zeros(1, 1, 1), ln, torch.zeros(1, 1, 4), 1, 4),
              lambda: fta.flash_cache_evict(c, torch.zeros(1, 1, 4), ln, 2)):
        with pytest.raises(ValueError, match="requires CUDA tensors"):
            f()


def test_what_is_written_lies_apart():
    """``out`` and the inputs of an eviction, and the weights and their cache, by address alone."""
    f16, f32 = torch.float16, torch.float32
    kv = (torch.Size((1, 4, 32)), (128, 32, 1), f16)
    w = (torch.Size((1, 2, 4)), (8, 4, 1), f32)
    metas, to_metas = (kv, kv, w), (kv, kv, tuple(w))
    apart = lambda at, to: cache_evict._check_apart("evict", False, metas, (kv, kv, (w[0], w[1], w[2])), at, to)  # noqa: E731
    apart((0, 256, 512), (1024, 1280, 1536))
    for to in ((1024, 1280, 1280 + 252), (1024, 1024, 2048), (1024, 1024 + 32, 2048), (240, 1280, 2048), (1024, 1280, 540)):
        with pytest.raises(ValueError):
            apart((0, 256, 512), to)
    assert to_metas is not metas


def test_position_offset_of_no_dimensions_is_a_number():
    """Only int32 [B] is an offset for each request; a tensor of no dimensions is a whole number, as any other is."""
    from flash_topk_attn_v2.qk_prep import offsets

    cpu = torch.device("cpu")
    for x in (5, 5.0, torch.tensor(5), torch.tensor(5, dtype=torch.int32)):
        assert offsets("x", x, 2, cpu, 64, 8) == (5, None)
    number, each = offsets("x", torch.tensor([3, 4], dtype=torch.int32), 2, cpu, 64, 8)
    assert number == 0 and each.tolist() == [3, 4]
    for x in (torch.tensor(0.5), torch.tensor([3], dtype=torch.int32), torch.tensor([3, 4]), torch.tensor([[3, 4]], dtype=torch.int32)):
        with pytest.raises(ValueError):
            offsets("x", x, 2, cpu, 64, 8)
