"""Infinite keys and values in a cache: a key scored -inf drops out, an infinite
value reaches the queries that see it and no other, and no weight turns to NaN."""
import math

import pytest
import torch

import _cachetight as tight
from fbsa_amd import cache
from test_gpu_cache import DEV, _ints, _make, _randn

pytestmark = pytest.mark.gpu


def _call(q, k, v, kp, vp, lens, **kw):
    if kp is None:
        return cache.cache_attention(q, k, v, _ints(lens), need_lse=True, **kw)
    return cache.shared_prefix_attention(q, kp, vp, k, v, _ints(lens), need_lse=True, **kw)


def _check(q, k, v, kp, vp, lens, g, count=None, gate=None):
    w = _randn(g, *k.shape[:3]).abs()
    out = w.clone()
    o, lse = _call(q, k, v, kp, vp, lens, count=_ints(count), weight=w, out_weight=out, out_gate=gate)
    r = tight.attend(q, k, v, lens, count, kp, vp, None, gate, w)
    rows = q.shape[2] * (q.shape[1] // k.shape[1])
    P = 0 if kp is None else kp.shape[1]
    rounded = rows > 16 or (P > 0 and q.shape[0] * rows > 16)
    tight.check((o, lse, out), r, q, k.shape[2] + P, rounded, gate is not None)
    return o, lse, out


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("T", [5, 7, 20, 41, 60])
def test_weights_beside_keys_scored_minus_infinity(dt, D, T):
    # 15, 21, 60, 123 and 180 rows: no whole number of the kernels' row tiles
    lens = [180, 61]
    q, k, v, _, _, g = _make(dt, 2, 6, 2, T, 180, D, lens)
    q[..., 3] = q[..., 3].abs() + 0.5
    for s in (0, 17, 59, 60, 150, 179):
        k[:, s % 2, s, 3] = -math.inf
    for b, n in enumerate(lens):
        k[b, :, n:] = math.nan
    _check(q, k, v, None, None, lens, g)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [8, 24, 40, 80, 136, 248])
@pytest.mark.parametrize("T,P", [(1, 0), (3, 45), (40, 0), (30, 70)])
def test_keys_scored_minus_infinity_at_head_dims_between(dt, D, T, P):
    # the last 16 bytes of a row hold the infinity
    lens = [170, 57]
    q, k, v, kp, vp, g = _make(dt, 2, 6, 2, T, 170, D, lens, P=P)
    q[..., D - 1] = q[..., D - 1].abs() + 0.5
    for s in (0, 31, 50, 169):
        k[:, s % 2, s, D - 1] = -math.inf
    for b, n in enumerate(lens):
        k[b, :, n:] = math.nan
    if P:
        kp[0, P // 2, D - 1] = -math.inf
    _check(q, k, v, kp, vp, lens, g, gate=_randn(g, *q.shape, dtype=q.dtype))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,P", [(1, 0), (4, 33), (40, 0), (150, 90)])
def test_rows_whose_every_key_is_scored_minus_infinity(dt, T, P):
    # as a row that sees nothing: 0, -inf, and no weight; the weights of the rest do not suffer
    lens = [200, 150]
    q, k, v, kp, vp, g = _make(dt, 2, 4, 2, T, 200, 64, lens, P=P)
    q[..., 0] = q[..., 0].abs() + 0.5
    k[0, 0, :200, 0] = -math.inf
    if P:
        kp[0, :, 0] = -math.inf
    o, lse, out = _check(q, k, v, kp, vp, lens, g)
    assert (lse[0, :2] == -math.inf).all() and (o[0, :2] == 0).all() and lse[0, 2:].isfinite().all()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 72, 128, 256])
@pytest.mark.parametrize("Hq,T,P", [(2, 1, 0), (4, 4, 0), (4, 3, 60), (6, 50, 0), (4, 80, 60)])
def test_infinite_values(dt, D, Hq, T, P):
    lens, count = [150, 81, 1], [T, max(1, T - 2), 1]
    q, k, v, kp, vp, g = _make(dt, 3, Hq, 2, T, 150, D, lens, P=P)
    place = [(0, 0, 149, 1, math.inf), (0, 1, 148, D - 1, -math.inf), (0, 0, 100, 0, math.inf), (0, 0, 70, 0, -math.inf),
             (1, 0, 80, 5, math.nan), (1, 1, 0, 7, math.inf), (2, 0, 0, 2, -math.inf)]
    plain = v.clone()
    for b, h, s, d, x in place:
        v[b, h, s, d], plain[b, h, s, d] = x, 0.0
    if P:
        vp[1, 31, 4], first = -math.inf, vp.clone()
        first[1, 31, 4] = 0.0
    gate = _randn(g, *q.shape, dtype=q.dtype)
    o, lse, out = _check(q, k, v, kp, vp, lens, g, count, gate)
    # every other output as if the infinities were zeros, bit for bit
    o0, lse0 = _call(q, k, plain, kp, first if P else None, lens, count=_ints(count), out_gate=gate)
    assert torch.equal(lse, lse0)
    fin = o.isfinite()
    assert torch.equal(o[fin], o0[fin])


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_one_row_of_infinite_values(dt):
    # p = 1 exactly
    q, k, v, _, _, g = _make(dt, 1, 2, 1, 1, 40, 64, [1])
    v[0, 0, 0, ::3], v[0, 0, 0, 1::3] = math.inf, -math.inf
    o = cache.cache_attention(q, k, v, _ints([1]))
    assert torch.equal(o, v[:, :, :1].expand(1, 2, 1, 64))


@pytest.mark.parametrize("Hq,T,Hkv,S", [(8, 1, 8, 9000), (16, 300, 2, 700)])
def test_infinite_values_in_one_of_many_shares(Hq, T, Hkv, S):
    # the other shares, tiles and sequences keep their bits
    q, k, v, _, _, g = _make("bf16", 2, Hq, Hkv, T, S, 128, [S, S - 77])
    want = cache.cache_attention(q, k, v, _ints([S, S - 77]))
    v[1, 0, S - 200, 9] = math.inf
    got = cache.cache_attention(q, k, v, _ints([S, S - 77]))
    t = torch.arange(T, device=DEV)
    sees = (S - 77 - T + t >= S - 200).view(1, T).expand(Hq // Hkv, T)
    assert torch.equal(got[1, :Hq // Hkv, :, 9] == math.inf, sees)
    got[1, :Hq // Hkv, :, 9] = torch.where(sees, want[1, :Hq // Hkv, :, 9], got[1, :Hq // Hkv, :, 9])
    assert torch.equal(got, want)
