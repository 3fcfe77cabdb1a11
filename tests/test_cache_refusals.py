"""What the cache operators refuse, on the host: nothing here launches."""
import ctypes

import pytest
import torch

from fbsa_amd import _lib, cache

DUMMY = 1 << 20  # never dereferenced: validation fails first


def _attn(**kw):
    d = _lib.CacheDesc()
    d.dtype, d.B, d.Hq, d.Hkv, d.T, d.S, d.P, d.D, d.scale = _lib.BF16, 2, 4, 2, 1, 128, 0, 64, 0.125
    d.sq[:] = d.so[:] = d.sog[:] = (256, 64, 64)
    d.sk[:] = d.sv[:] = (2 * 128 * 64, 128 * 64, 64)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return d


def _call(d, weight=None, out_weight=None, ws=DUMMY, nbytes=1 << 40, q=DUMMY, kp=None, lens=DUMMY):
    return _lib.load().fbsa_cache_attn(d, q, DUMMY, DUMMY, lens, None, kp, kp, None, DUMMY, None, weight, out_weight, ws, nbytes, None)


def test_struct_layouts():
    assert ctypes.sizeof(_lib.AppendDesc) == 8 + 5 * 8 + 14 * 8
    assert ctypes.sizeof(_lib.CacheDesc) == 8 + 7 * 8 + 8 + 23 * 8
    assert ctypes.sizeof(_lib.EvictDesc) == 8 + 8 * 8 + 16 * 8


@pytest.mark.parametrize("kw,needle", [
    ({"dtype": 5}, "dtype"), ({"flags": 2}, "flags"), ({"T": 0}, "positive"), ({"S": 0}, "positive"), ({"P": -1}, "positive"),
    ({"Hkv": 3}, "multiple"), ({"D": 60}, "head dim"), ({"D": 264}, "head dim"), ({"scale": float("nan")}, "scale"),
    ({"S": 1 << 31}, "32-bit"), ({"B": 40000}, "grid"), ({"sk": (8192, 4096, 63)}, "stride"), ({"sv": (8192, -64, 64)}, "stride"),
    ({"sk": (0, 0, 1 << 26)}, "64 MiB"), ({"B": 64, "T": 1 << 19}, "grid"), ({"P": 8, "skp": (512, 60)}, "k_prefix"),
])
def test_attention_descriptor(kw, needle):
    lib = _lib.load()
    assert lib.fbsa_cache_attn_workspace_bytes(_attn(**kw)) == 0
    assert needle in lib.fbsa_last_error().decode()
    assert _call(_attn(**kw)) in (_lib.EINVAL, _lib.EUNSUPPORTED)


def test_attention_pointers_and_workspace():
    lib = _lib.load()
    d = _attn()
    need = lib.fbsa_cache_attn_workspace_bytes(d)
    assert need > 0
    assert _call(d, q=None) == _lib.EINVAL and _call(d, lens=None) == _lib.EINVAL
    assert _call(d, q=DUMMY + 8) == _lib.EINVAL and b"aligned" in lib.fbsa_last_error()
    assert _call(d, weight=DUMMY) == _lib.EINVAL and b"out_weight" in lib.fbsa_last_error()
    assert _call(d, out_weight=DUMMY) == _lib.EINVAL and b"FBSA_CACHE_WEIGHT" in lib.fbsa_last_error()
    assert _call(_attn(flags=_lib.CACHE_WEIGHT)) == _lib.EINVAL
    assert _call(d, ws=None) == _lib.EWORKSPACE and _call(d, nbytes=need - 1) == _lib.EWORKSPACE
    assert _call(d, ws=DUMMY + 128, nbytes=need) == _lib.EINVAL
    assert _call(_attn(P=16, skp=(1024, 64), svp=(1024, 64))) == _lib.EINVAL  # a prefix of no tensors
    assert lib.fbsa_cache_attn_workspace_bytes(None) == 0


def _evict(**kw):
    d = _lib.EvictDesc()
    d.dtype, d.B, d.H, d.S, d.SO, d.D, d.budget, d.recent, d.sink = _lib.BF16, 1, 2, 128, 64, 64, 64, 8, 4
    for s in ("sk", "sv", "sko", "svo"):
        getattr(d, s)[:] = (2 * 128 * 64, 128 * 64, 64)
    d.sw[:] = d.swo[:] = (256, 128)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,needle", [
    ({"dtype": -1}, "dtype"), ({"flags": 2}, "flags"), ({"budget": 0}, "positive"), ({"recent": 61}, "budget"),
    ({"sink": -1}, "budget"), ({"SO": 63}, "capacity"), ({"D": 4}, "head dim"), ({"B": 70000}, "grid"),
    ({"D": 256, "S": 1 << 28, "SO": 1 << 28, "budget": 1 << 28}, "grid"),
    ({"sko": (0, 0, 7)}, "stride"), ({"flags": 1}, "not the inputs"),
])
def test_evict_descriptor(kw, needle):
    p = [DUMMY * i for i in range(1, 9)]
    assert _lib.load().fbsa_cache_evict(_evict(**kw), *p[:4], *p[4:], DUMMY * 9, None, 0, None) in (_lib.EINVAL, _lib.EUNSUPPORTED)
    assert needle in _lib.load().fbsa_last_error().decode()


def test_evict_pointers():
    lib, p = _lib.load(), [DUMMY * i for i in range(1, 10)]
    assert lib.fbsa_cache_evict(_evict(), *p[:3], None, *p[4:], None, 0, None) == _lib.EINVAL
    assert lib.fbsa_cache_evict(_evict(), *p[:4], p[0], *p[5:], None, 0, None) == _lib.EINVAL and b"overlap" in lib.fbsa_last_error()
    assert lib.fbsa_cache_evict(_evict(), *p[:8], p[3], None, 0, None) == _lib.EINVAL and b"new_lens" in lib.fbsa_last_error()
    assert lib.fbsa_cache_evict_workspace_bytes(_evict()) == 0
    d = _evict(S=40000)
    need = lib.fbsa_cache_evict_workspace_bytes(d)
    assert need > 0 and lib.fbsa_cache_evict(d, *p, DUMMY, need - 1, None) == _lib.EWORKSPACE
    assert lib.fbsa_cache_evict(d, *p, None, 0, None) == _lib.EWORKSPACE
    assert lib.fbsa_cache_evict(d, *p, DUMMY + 16, need, None) == _lib.EINVAL
    # in place: room for the rows' way, a part of them at a time
    size = lambda **kw: lib.fbsa_cache_evict_workspace_bytes(_evict(flags=1, **kw))
    assert size(S=16384, SO=16384, budget=512) == 0 and 0 < size(S=16384, SO=16384, budget=16383) <= 64 << 20
    d = _evict(flags=1, S=16384, SO=16384, budget=4096)
    same = [p[0], p[1], p[2], p[3], p[0], p[1], p[2], p[7], p[8]]
    assert lib.fbsa_cache_evict(d, *same, None, 0, None) == _lib.EWORKSPACE


@pytest.mark.parametrize("kw,needle", [({"T": 0}, "positive"), ({"D": 12}, "head dim"), ({"flags": 1}, "flags"),
                                       ({"skn": (1, 1, 1)}, "stride"), ({"B": 1 << 20, "H": 1 << 20}, "grid"), ({"B": 1 << 14, "H": 1 << 7, "T": 300}, "grid")])
def test_append_descriptor(kw, needle):
    d = _lib.AppendDesc()
    d.dtype, d.B, d.H, d.T, d.S, d.D = _lib.BF16, 1, 2, 1, 16, 64
    for s in ("sk", "sv", "skn", "svn"):
        getattr(d, s)[:] = (2048, 1024, 64)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    assert _lib.load().fbsa_cache_append(d, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, None, None, None) in (_lib.EINVAL, _lib.EUNSUPPORTED)
    assert needle in _lib.load().fbsa_last_error().decode()


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    lens = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: cache.cache_attention(x, x, x, lens), lambda: cache.append(x, x, x, x, lens),
                 lambda: cache.shared_prefix_attention(x, x[0], x[0], x, x, lens),
                 lambda: cache.evict(x, x, torch.zeros(1, 2, 8), lens, 4)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_written_tensors_must_not_overlap_themselves():
    x = torch.zeros(2, 8, 16)
    cache._written("t", "x", x)
    cache._written("t", "x", x.transpose(0, 1)[:, ::2])
    cache._written("t", "x", torch.zeros(1, 8).expand(1, 8))
    with pytest.raises(ValueError, match="overlap"):
        cache._written("t", "x", torch.zeros(1, 16).expand(2, 16))
    with pytest.raises(ValueError, match="overlap"):
        cache._written("t", "x", x.as_strided((2, 8, 16), (64, 16, 1)))
    with pytest.raises(ValueError, match="reads"):
        cache._apart("t", ((64, 64),), ((0, 8), (120, 200)))
    with pytest.raises(ValueError, match="same buffer"):
        cache._apart("t", ((64, 64), (64, 32)), ())
    cache._apart("t", ((64, 64), (128, 64)), ((0, 64), (192, 8)))
    assert cache._bytes(x[0, 4:]) == 4 * 16 * 4 and cache._bytes(x[:, :, :1]) == (8 * 16 + 7 * 16 + 1) * 4


def test_plans_follow_layouts_not_addresses():
    def key(*ts):
        return hash(cache._key("t", (1, None), ts))
    x = torch.zeros(2, 8, 16)
    assert key(x, None) == key(torch.ones(2, 8, 16), None)
    assert key(x) != key(x.half()) and key(x) != key(x.transpose(0, 1)) and key(x, x) != key(x, None)
