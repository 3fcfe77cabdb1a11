"""Cache attention at the sizes that choose each way of computing it, against 64
bits: tiles that write their results themselves, tiles of prefix and own rows in
launches of their own, the most parts that are joined, far-apart rows."""
import ctypes

import pytest
import torch

import _cachetight as tight
from fbsa_amd import _lib, cache
from test_gpu_cache import DEV, DT, _gen, _ints, _make, _randn

pytestmark = pytest.mark.gpu


def _workspace(q, k, P, weight):
    d = _lib.CacheDesc()
    d.dtype = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}[q.dtype]
    d.B, d.Hq, d.T, d.D = q.shape
    d.Hkv, d.S, d.P, d.scale, d.flags = k.shape[1], k.shape[2], P, 0.125, _lib.CACHE_WEIGHT if weight else 0
    return _lib.load().fbsa_cache_attn_workspace_bytes(ctypes.byref(d))


def _run(dt, B, Hq, Hkv, T, S, D, lens, count=None, P=0, weight=True, direct=False, seed=0):
    q, k, v, kp, vp, g = _make(dt, B, Hq, Hkv, T, S, D, lens, seed, P)
    gate = _randn(g, B, T, Hq, D, dtype=q.dtype).transpose(1, 2)
    w = _randn(g, B, Hkv, S).abs() if weight else None
    out = torch.full_like(w, -7.0) if weight else None
    parts = 4 * B * Hq * T * D     # bytes of one fp32 part of every row: a call that joins any holds them
    assert (_workspace(q, k, P, False) < parts) == direct
    kw = dict(count=_ints(count), out_gate=gate, weight=w, out_weight=out, need_lse=True)
    if P:
        o, lse = cache.shared_prefix_attention(q, kp, vp, k, v, _ints(lens), **kw)
    else:
        o, lse = cache.cache_attention(q, k, v, _ints(lens), **kw)
    if weight:
        for b, n in enumerate(lens):
            assert (out[b, :, n:] == -7.0).all()
            out[b, :, n:] = w[b, :, n:]
    rows = T * (Hq // Hkv)
    r = tight.attend(q, k, v, lens, count, kp, vp, None, gate, w)
    tight.check((o, lse, out), r, q, S + P, rows > 16 or (P > 0 and B * rows > 16), True)


@pytest.mark.parametrize("dt,S", [("bf16", 128), ("fp16", 100), ("fp32", 32)])
@pytest.mark.parametrize("D", [32, 40, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,T", [(4, 2, 25), (3, 1, 27), (8, 2, 40), (7, 1, 50)])
def test_one_share_writes_its_results(dt, S, D, Hq, Hkv, T):
    # tiles of 64, 96 (six waves), 80 and 128 rows; weights of up to 128 rows and of more
    _run(dt, 3, Hq, Hkv, T, S, D, [S, S // 2, 3], count=[T, T - 4, min(T, 9)], direct=True)


@pytest.mark.parametrize("dt,B,Hq,Hkv,T,S,D", [("bf16", 1, 260, 260, 70, 330, 256), ("fp16", 1, 520, 520, 65, 300, 64),
                                               ("fp32", 1, 260, 130, 50, 150, 256), ("bf16", 3, 700, 700, 17, 270, 32)])
def test_one_share_of_several_chunks(dt, B, Hq, Hkv, T, S, D):
    # enough tiles to fill the card: each goes through all its keys
    lens = [S, S - 64, S - 65][:B]
    _run(dt, B, Hq, Hkv, T, S, D, lens, direct=True)


def test_one_share_of_a_long_chunk():
    # a prompt's chunk: 256 tiles of 128 rows, weights of more than 128 rows
    _run("bf16", 1, 16, 2, 2048, 2300, 256, [2290], direct=True)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("T,S", [(40, 350), (257, 300), (300, 1000)])
def test_weights_of_many_rows_in_fp16(D, T, S):
    _run("fp16", 2, 8, 2, T, S, D, [S, S - 51], count=[T, T - 30])


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("fp16", 128), ("bf16", 256)])
def test_prefix_and_own_tiles_in_launches_of_their_own(dt, D):
    # 640 own tiles of 32 rows and a prefix's tiles of 128: workgroups of other sizes
    B, T = 40, 10
    _run(dt, B, 48, 16, T, 140, D, [T + 3 * b for b in range(B)], P=150)


@pytest.mark.parametrize("dt,S", [("bf16", 20000), ("fp16", 17000), ("fp32", 8300)])
@pytest.mark.parametrize("n", [None, 700])
def test_the_most_parts(dt, S, n):
    # 256 shares of the prefix and 256 of the own rows; a short sequence leaves most of the latter empty
    _run(dt, 1, 2, 1, 1, S, 64, [S if n is None else n], P=S + 33)


@pytest.mark.parametrize("T,P", [(1, 0), (20, 0), (20, 1)])
def test_rows_almost_64_mib_apart(T, P):
    # offsets within a chunk of 64 rows pass 2^31
    g, S, D, step = _gen(4), 130, 64, (1 << 25) - 8
    big = torch.empty(S * step, dtype=torch.bfloat16, device=DEV)
    k, v = (big.as_strided((1, 1, S, D), (S * step, S * step, step, 1), at) for at in (0, 4096))
    k.copy_(_randn(g, 1, 1, S, D))
    v.copy_(_randn(g, 1, 1, S, D))
    near = [x.contiguous() for x in (k, v)]
    q = _randn(g, 1, 2, T, D, dtype=torch.bfloat16)
    far_w, near_w = (torch.zeros(1, 1, S, device=DEV) for _ in range(2))
    kw = dict(need_lse=True)
    if P:
        far = cache.shared_prefix_attention(q, k[0], v[0], k, v, _ints([S]), out_weight=far_w, **kw)
        want = cache.shared_prefix_attention(q, near[0][0], near[1][0], *near, _ints([S]), out_weight=near_w, **kw)
    else:
        far = cache.cache_attention(q, k, v, _ints([S]), out_weight=far_w, **kw)
        want = cache.cache_attention(q, *near, _ints([S]), out_weight=near_w, **kw)
    assert all(torch.equal(x, y) for x, y in zip((*far, far_w), (*want, near_w)))
    assert want[0].isfinite().all() and DT["bf16"] == want[0].dtype
