"""The cache operators' host side: what is refused before a launch, workspaces,
64-bit lengths, forward-mode gradients."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw

import _cachetight as tight
from fbsa_amd import _lib, cache


def _desc(**kw):
    d = _lib.CacheDesc()
    d.dtype, d.B, d.Hq, d.Hkv, d.T, d.S, d.P, d.D, d.scale = _lib.BF16, 1, 1, 1, 1, 128, 0, 64, 0.125
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _bytes(**kw):
    return _lib.load().fbsa_cache_attn_workspace_bytes(ctypes.byref(_desc(**kw)))


def test_lengths_beyond_32_bits_are_clamped_not_wrapped():
    x = torch.tensor([1 << 32, (1 << 32) + 5, -(1 << 40), 7, -3, (1 << 31) - 1], dtype=torch.int64)
    assert cache._int32(x).tolist() == [(1 << 31) - 1, (1 << 31) - 1, -(1 << 31), 7, -3, (1 << 31) - 1]
    assert cache._int32(x).dtype == torch.int32 and cache._int32(None) is None
    y = torch.tensor([1, 2, 3, 4], dtype=torch.int32)
    assert cache._int32(y) is y and cache._int32(y[::2]).tolist() == [1, 3] and cache._int32(y[::2]).is_contiguous()


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_gradients_are_refused(grad):
    x = torch.zeros(1, 2, 8, 64)
    with fw.dual_level(), torch.set_grad_enabled(grad):
        cache._key("t", (), (x, None))
        dual = fw.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="gradients"):
            cache._key("t", (), (x, dual))


@pytest.mark.parametrize("kw", [
    dict(dtype=_lib.F32, S=(1 << 30) + (1 << 20), D=8, T=129, flags=_lib.CACHE_WEIGHT),   # 128 keys of 512 threads each
    dict(B=65535, S=1 << 28, D=8, flags=_lib.CACHE_WEIGHT),                               # 1024 keys of 256 threads each
])
def test_launches_of_more_than_32_bits_of_threads_are_refused(kw):
    assert _bytes(**kw) == 0 and b"grid" in _lib.load().fbsa_last_error()
    assert _bytes(**{**kw, "S": 1 << 16}) > 0
    assert _bytes(**{**kw, "flags": 0}) > 0


@pytest.mark.parametrize("scale", [3e38, -3e38, float("inf"), float("nan")])
def test_scales_that_overflow_the_exponent_are_refused(scale):
    # x = scale q.k goes through exp2, its scale times log2(e): 2.36e38 is the largest that stays finite
    assert _bytes(scale=scale) == 0 and b"scale" in _lib.load().fbsa_last_error()
    assert _bytes(scale=2.3e38) > 0 and _bytes(scale=-2.3e38) > 0 and _bytes(scale=0.0) > 0


@pytest.mark.parametrize("kw", [dict(B=32, Hq=32, Hkv=8, T=1024, S=8192, D=256), dict(B=16, Hq=64, Hkv=8, T=2048, S=4096, D=128)])
def test_tiles_that_write_their_results_need_no_parts(kw):
    assert 0 < _bytes(**kw) <= 256
    # with weights: the rows' normalisers
    rows = kw["B"] * kw["Hq"] * kw["T"]
    assert 4 * rows <= _bytes(**kw, flags=_lib.CACHE_WEIGHT) <= 4 * rows + 4096
    assert _bytes(**kw, P=64) > 4 * rows * kw["D"]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rounded", [False, True])
def test_the_bounds_pass_a_rounded_result_and_see_a_missing_key(dt, rounded):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 2, n, 64, generator=g).to(dt) for n in (40, 1000, 1000))
    lens = [1000]
    r = tight.attend(q, k, v, lens, weight=torch.zeros(1, 2, 1000))
    tight.check((r["o"].to(dt), r["lse"].float(), r["w"].float()), r, q, 1000, rounded)
    less = v.clone()
    less[0, 1, 500] = 0   # one of a thousand values left out, of one head
    o = tight.attend(q, k, less, lens)["o"].to(dt)
    with pytest.raises(AssertionError, match="bound"):
        tight.check((o, r["lse"].float(), None), r, q, 1000, rounded)
