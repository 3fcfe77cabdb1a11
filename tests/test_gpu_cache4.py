"""A cache in 4 bits on the GPU: rows written, read back and attended, against 64 bits."""
import math
import threading

import numpy as np
import pytest
import torch

import _cache4ref as ref
from fbsa_amd import cache, cache4

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)


def _held(g, dt, B, H, S, D):
    """A cache of random codes and steps as rows of size 1 have them (NaN nowhere)."""
    k4, v4 = (torch.randint(0, 256, (B, H, S, D // 2), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2))
    step = (0.2 + 0.3 * torch.rand(B, H, S, 2, -(-D // 64), generator=g, device=DEV)).mul(64).round().div(64)
    return k4, v4, step.to(ref.step_type(dt))


# ---- writing and reading -------------------------------------------------------
def _rows(kind, g, dt, *shape):
    x = _randn(g, *shape)
    big, small = (15, -24) if dt == torch.float16 else (127, -126)
    if kind == "wide":          # every size that the type has, a row at a time
        x = x * torch.exp2(torch.randint(small, big, (*shape[:-1], 1), generator=g, device=DEV).float())
    elif kind == "ties":        # on and beside the borders between codes, for steps of few bits
        border = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0], device=DEV)
        x = border[torch.randint(0, 14, shape, generator=g, device=DEV)]
        x = x * (1 - 2 * torch.randint(0, 2, shape, generator=g, device=DEV))
        x[..., ::64] = 6.0
        if dt == torch.float32:
            x = x * (1 + torch.randint(-1, 2, shape, generator=g, device=DEV) * 2.0 ** -23)
        x = x * torch.randint(1, 32, (*shape[:-1], 1), generator=g, device=DEV) * 2.0 ** -6
    elif kind == "steps":       # largest magnitudes on and beside the ties of the step's rounding
        x = x.clamp(-1, 1) * 0.01
        top = 6 * (torch.randint(64, 128, (*shape[:-1], 1), generator=g, device=DEV) + 0.0)
        x[..., :1] = top * (1 + torch.randint(-1, 2, top.shape, generator=g, device=DEV) * 2.0 ** -23)
    elif kind == "edge":        # zeros, the type's largest and smallest numbers
        top, low = torch.finfo(dt).max, torch.finfo(dt).smallest_normal
        pool = torch.tensor([0.0, -0.0, top, -top, low, -low, low / 8, 1.0, 6.5 * low, 100 * low], device=DEV)
        pick = torch.randint(0, 10, (*shape[:-1], 1), generator=g, device=DEV)
        x = pool[pick] * torch.randint(-1, 2, shape, generator=g, device=DEV).float()
    x = x.to(dt)
    return torch.where(x.isfinite(), x, torch.sign(x) * torch.finfo(dt).max)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("kind", ["normal", "wide", "ties", "steps", "edge"])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 224, 256])
def test_rows_written_and_read_back(dt, kind, D):
    g, dt, B, H, T = _gen(D), DT[dt], 2, 3, 57
    k, v = _rows(kind, g, dt, B, H, T, D), _rows("normal" if kind == "edge" else kind, g, dt, B, H, T, D)
    held = cache4.empty(B, H, T + 8, D, dtype=dt)
    cache4.append(*held, k, v, _ints([0, 5]))
    want = ref.held(k, v)
    got = ref.values(held)
    for x, y, s, n in zip(want, got, (k, v), range(2)):
        for b, at in enumerate((0, 5)):
            assert torch.equal(x[b], y[b, :, at:at + T]), f"{'kv'[n]} of sequence {b}"
            assert torch.equal(torch.from_numpy(ref.steps(s)[b]), held[2][b, :, at:at + T, n].cpu().double())
    # the rows come back exactly, in every type that holds them
    for as_type in {dt, torch.float16 if dt == torch.float16 else torch.float32}:
        if dt == torch.float16 and as_type != dt:
            continue
        back = cache4.read(*held, _ints([0, 5]), T, dtype=as_type)
        assert all(torch.equal(x.cpu().double(), y) for x, y in zip(back, want))
    if dt == torch.float32:  # (32-bit rows are held as bf16 numbers too)
        back = cache4.read(*held, _ints([0, 5]), T, dtype=torch.bfloat16)
        assert all(torch.equal(x.cpu().double(), y) for x, y in zip(back, want))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D", [32, 96, 256])
def test_rows_that_are_not_finite_are_nan(dt, D):
    g, dt = _gen(1), DT[dt]
    k, v = (_randn(g, 2, 2, 9, D, dtype=dt) for _ in range(2))
    k[0, 0, 2, D - 1], k[0, 1, 4, 0], v[1, 0, 6, 5], v[1, 1, 8, D // 2] = math.nan, math.inf, -math.inf, math.nan
    held = cache4.empty(2, 2, 9, D, dtype=dt)
    cache4.append(*held, k, v, _ints([0, 0]))
    back = cache4.read(*held, None, 9, dtype=dt)
    bad = torch.zeros(2, 2, 9, dtype=torch.bool)
    bad[0, 0, 2] = bad[0, 1, 4] = bad[1, 0, 6] = bad[1, 1, 8] = True
    for x, y in zip(back, ref.held(k, v)):
        x = x.cpu().double()
        assert torch.equal(x.isnan(), bad.unsqueeze(-1).expand_as(x)) and torch.equal(x.nan_to_num(0), y.nan_to_num(0))


@pytest.mark.parametrize("dt", list(DT))
def test_only_the_given_rows_change(dt):
    g, dt, B, H, S, D, T = _gen(3), DT[dt], 5, 2, 40, 64, 12
    k, v = (_randn(g, B, T, H, D, dtype=dt).transpose(1, 2) for _ in range(2))   # rows of a strided projection
    held = _held(g, dt, B, H, S, D)
    before = [x.clone() for x in held]
    start, count = [0, 33, -4, 45, 7], [12, 12, 12, 12, 3]
    cache4.append(*held, k, v, _ints(start), count=_ints(count))
    kept = torch.ones(B, S, dtype=torch.bool)
    want = ref.held(k, v)
    got = ref.values(held)
    for b in range(B):
        for t in range(T):
            at = start[b] + t
            if t < count[b] and 0 <= at < S:
                kept[b, at] = False
                assert all(torch.equal(x[b, :, at], y[b, :, t]) for x, y in zip(got, want))
    for x, y in zip(held, before):
        for b in range(B):
            assert torch.equal(x[b][:, kept[b].to(DEV)], y[b][:, kept[b].to(DEV)])


@pytest.mark.parametrize("dt", list(DT))
def test_reading_outside_and_into_other_layouts(dt):
    g, dt, B, H, S, D, T = _gen(4), DT[dt], 5, 2, 40, 160, 23
    held = _held(g, dt, B, H, S, D)
    first, count = [0, 30, -5, 60, 3], [23, 23, 23, 23, 0]
    both = ref.values(held)
    out = tuple(torch.full((B, T, H, D), 9.0, dtype=dt, device=DEV).transpose(1, 2) for _ in range(2))
    got = cache4.read(*held, _ints(first), T, count=_ints(count), out=out)
    assert got[0] is out[0] and got[1] is out[1]
    for x, y in zip(got, both):
        for b in range(B):
            for t in range(T):
                at = first[b] + t
                want = y[b, :, at] if t < count[b] and 0 <= at < S else torch.zeros(H, D, dtype=torch.float64)
                assert torch.equal(x[b, :, t].cpu().double(), want)
    alone = cache4.read(*held, _ints(first), T, count=_ints(count), dtype=dt)
    assert all(torch.equal(x, y) for x, y in zip(alone, got))
    # (64-bit places beyond 32 bits are far out, not wrapped)
    far = torch.tensor([1 << 32, -(1 << 40), 1 << 33, 0, 5], device=DEV)
    x = cache4.read(*held, far, 1, dtype=dt)[0]
    assert (x[:3] == 0).all() and torch.equal(x[3, :, 0].cpu().double(), both[0][3, :, 0])


def test_rows_in_interleaved_buffers():
    """Codes of keys and values side by side in one buffer, heads inside rows, steps of an odd number of rows."""
    g, B, H, S, D = _gen(5), 2, 3, 77, 64
    both = torch.zeros(B, S, H, 2, D // 2, dtype=torch.uint8, device=DEV)
    k4, v4 = both[..., 0, :].transpose(1, 2), both[..., 1, :].transpose(1, 2)
    step = torch.zeros(B, H, S, 2, 1, dtype=torch.bfloat16, device=DEV)
    k, v = (_randn(g, B, H, S, D, dtype=torch.bfloat16) for _ in range(2))
    cache4.append(k4, v4, step, k, v, _ints([0, 0]))
    plain = cache4.empty(B, H, S, D)
    cache4.append(*plain, k, v, _ints([0, 0]))
    assert torch.equal(k4, plain[0]) and torch.equal(v4, plain[1]) and torch.equal(step, plain[2])
    q = _randn(g, B, 2 * H, 1, D, dtype=torch.bfloat16)
    got = [cache4.cache_attention(q, *x, _ints([77, 5]), need_lse=True) for x in ((k4, v4, step), plain)]
    assert all(torch.equal(x, y) for x, y in zip(*got))
    ref.check_attend(got[0], plain, q, [77, 5])


# ---- attention -----------------------------------------------------------------
def _attend(dt, B, Hq, Hkv, T, S, D, lens, count=None, scale=None, gated=False, seed=0):
    g, dt = _gen(seed), DT[dt]
    held = _held(g, dt, B, Hkv, S, D)
    q = _randn(g, B, T, Hq, D, dtype=dt).transpose(1, 2)
    gate = _randn(g, B, T, Hq, D, dtype=dt).transpose(1, 2) if gated else None
    got = cache4.cache_attention(q, *held, _ints(lens), count=_ints(count), scale=scale, out_gate=gate, need_lse=True)
    ref.check_attend(got, held, q, lens, count, scale, gate)
    return got, held, q


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("Hq,Hkv,T", [(2, 2, 1), (6, 2, 1), (4, 1, 1), (5, 1, 1), (8, 1, 2), (4, 2, 3), (8, 2, 5), (16, 2, 9), (2, 2, 130)])
def test_attention(dt, D, Hq, Hkv, T):
    lens = [333, 64, max(T, 65)]
    _attend(dt, 3, Hq, Hkv, T, 400, D, lens, count=[T, max(1, T - 2), T], gated=True, seed=D + T)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("Hq,Hkv,T", [(1, 1, 1), (8, 1, 1), (4, 1, 20)])
@pytest.mark.parametrize("S", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129])
def test_lengths_about_a_chunk(dt, D, Hq, Hkv, T, S):
    lens = [S, S - 1, S // 2, 0]
    _attend(dt, 4, Hq, Hkv, T, S, D, lens, seed=S)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("Hq,Hkv,T", [(1, 1, 1), (6, 1, 2), (4, 2, 40)])
def test_rows_that_see_nothing(dt, Hq, Hkv, T):
    """Lengths below the new tokens', of zero, negative and beyond the capacity; counts of
    zero, negative and beyond T."""
    lens, count = [0, -7, 1, 500, 90, 90, 3], [T, T, T, T, 0, -3, T + 9]
    got, _, _ = _attend(dt, 7, Hq, Hkv, T, 90, 64, lens, count, gated=True)
    o, lse = got
    assert (o[[0, 1, 4, 5]] == 0).all() and (lse[[0, 1, 4, 5]] == -math.inf).all()


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("scale", [0.0, -0.1, 0.3])
@pytest.mark.parametrize("Hq,T", [(1, 1), (16, 1), (4, 30)])
def test_scales(dt, scale, Hq, T):
    _attend(dt, 1, Hq, 1, T, 200, 128, [150], scale=scale)


@pytest.mark.parametrize("dt,Hq,Hkv,T,S,D", [("bf16", 8, 8, 1, 20000, 64), ("fp16", 16, 2, 1, 9000, 256), ("fp32", 4, 4, 1, 7001, 64),
                                             ("bf16", 32, 8, 1, 5000, 128), ("bf16", 16, 2, 300, 2500, 256), ("fp32", 8, 8, 40, 3001, 96),
                                             ("fp16", 16, 2, 5, 6000, 128)])
def test_many_shares(dt, Hq, Hkv, T, S, D):
    _attend(dt, 2, Hq, Hkv, T, S, D, [S, S // 3], gated=True)


@pytest.mark.parametrize("dt,B,Hq,Hkv,T,S,D", [("bf16", 70, 2, 2, 1, 900, 64), ("fp16", 150, 4, 1, 2, 700, 32), ("fp32", 65, 1, 1, 1, 6000, 64),
                                               ("bf16", 200, 8, 1, 3, 300, 128), ("fp16", 67, 16, 1, 4, 400, 64), ("bf16", 1100, 8, 8, 1, 90, 32),
                                               ("bf16", 8300, 1, 1, 1, 66, 32)])
def test_many_sequences(dt, B, Hq, Hkv, T, S, D):
    """More sequences than a wave has lanes, of all lengths, some without new tokens."""
    lens = [(37 * b * b) % (S + 1) for b in range(B)]
    count = [(b * 7) % (T + 1) if b % 3 == 0 else T for b in range(B)]
    _attend(dt, B, Hq, Hkv, T, S, D, lens, count, seed=B)


@pytest.mark.parametrize("dt,B,Hq,Hkv,T,S,D", [("bf16", 2, 8, 1, 900, 5000, 64), ("fp32", 2, 8, 1, 700, 3000, 32), ("fp16", 3, 4, 1, 500, 9000, 128),
                                               ("bf16", 3, 2, 1, 300, 4000, 256), ("fp32", 3, 2, 2, 200, 2500, 160), ("bf16", 100, 8, 1, 5, 1500, 256),
                                               ("fp16", 200, 8, 1, 6, 700, 192), ("bf16", 1100, 8, 1, 4, 200, 256)])
def test_many_tiles(dt, B, Hq, Hkv, T, S, D):
    """Tiles of many rows, more of them than a wave has lanes or than the card runs, whose
    sequences differ in length and whose last tiles may be padding."""
    lens = [S, 40, (S * 2) // 3][:B] + [(53 * b * b) % (S + 1) for b in range(3, B)]
    count = [T, T // 3, T - 1][:B] + [(b * 5) % (T + 1) for b in range(3, B)]
    _attend(dt, B, Hq, Hkv, T, S, D, lens, count, seed=T)


@pytest.mark.parametrize("dt,B,Hq,Hkv,T,S,D", [("bf16", 16, 8, 1, 300, 9000, 128), ("fp16", 5, 8, 1, 450, 6000, 256), ("fp32", 40, 4, 2, 300, 3000, 32),
                                               ("bf16", 3, 16, 4, 520, 5000, 64), ("fp32", 9, 2, 1, 900, 2500, 224)])
def test_one_long_sequence(dt, B, Hq, Hkv, T, S, D):
    """Tiles in several pieces beside tiles in one, and tiles that see nothing."""
    lens = [(29 * b) % 200 for b in range(B)]
    count = [T if b % 4 else T // 2 for b in range(B)]
    lens[1], count[1] = S, T
    _attend(dt, B, Hq, Hkv, T, S, D, lens, count, seed=B, gated=dt != "fp32")


@pytest.mark.parametrize("dt,B,H,T,S,D", [("bf16", 40, 256, 20, 600, 32), ("fp16", 18, 256, 40, 300, 32), ("fp32", 20, 256, 4, 250, 160)])
def test_one_long_sequence_of_more_than_run_at_a_time(dt, B, H, T, S, D):
    """So many heads that the card goes through the sequences several times, which are cut all the same."""
    lens = [(29 * b) % 100 for b in range(B)]
    count = [T if b % 4 else T // 2 for b in range(B)]
    lens[1], count[1] = S, T
    _attend(dt, B, H, H, T, S, D, lens, count, seed=B)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("Hq,T", [(1, 1), (8, 1), (16, 1), (8, 3), (8, 12), (8, 30)])
def test_small_and_large_rows(dt, Hq, T):
    """Steps near the ends of what a type holds (fp16: subnormal values)."""
    g, t = _gen(T), DT[dt]
    held = _held(g, t, 1, 1, 200, 64)
    # (32-bit pieces are exact down to 2^-126, 24 bits below a probability times a step)
    small, big = (2.0 ** -23, 512.0) if t == torch.float16 else (2.0 ** -60, 2.0 ** 100)
    q = _randn(g, 1, Hq, T, 64, dtype=t)
    for size in (small, big):
        step = held[2].clone()
        step[:, :, :, 1] = (step[:, :, :, 1].float() * 32).round().to(step.dtype) * size   # (of few bits: exact)
        got = cache4.cache_attention(q, held[0], held[1], step, _ints([190]), need_lse=True)
        ref.check_attend(got, (held[0], held[1], step), q, [190])


def test_rows_beyond_4_gib():
    """Codes of more than 2^32 bytes: rows behind them are written, read and attended."""
    S, D = (1 << 26) + 1000, 128
    held = cache4.empty(1, 1, S, D)
    g = _gen(0)
    k, v = (_randn(g, 1, 1, 5, D, dtype=torch.bfloat16) for _ in range(2))
    k[0, 0, 4] = 4.0
    for at in (S - 5, S - 1003):
        cache4.append(*held, k, v, _ints([at]))
        want = ref.held(k, v)
        assert all(torch.equal(x.cpu().double(), y) for x, y in zip(cache4.read(*held, _ints([at]), 5), want))
    # (the others' keys are zeros: a query along the last row's key has all its weight there)
    q = torch.full((1, 1, 1, D), 2.0, dtype=torch.bfloat16, device=DEV)
    o = cache4.cache_attention(q, *held, _ints([S]))
    both = want[1][0, 0, 4]   # two such rows, of the same value
    assert (o[0, 0, 0].cpu().double() - both).abs().max() <= 2.0 ** -8 * both.abs().max() + 1e-6
    many = cache4.cache_attention(q.expand(1, 1, 40, D).contiguous(), *held, _ints([S]))
    assert (many[0, 0, -1].cpu().double() - both).abs().max() <= 2.0 ** -7 * both.abs().max() + 1e-6


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("Hq,T", [(1, 1), (8, 1), (2, 12)])
def test_heavy_keys(dt, Hq, T):
    """Scores far apart: one key holds nearly all of a query's weight, the running maximum moves."""
    g, t = _gen(9), DT[dt]
    held = _held(g, t, 1, 1, 300, 64)
    held[2][:, :, ::37, 0] *= 8
    q = 4 * _randn(g, 1, Hq, T, 64, dtype=t)
    got = cache4.cache_attention(q, *held, _ints([300]), need_lse=True)
    ref.check_attend(got, held, q, [300])


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,T", [(2, 2, 4), (8, 2, 4), (4, 2, 30)])
def test_nan_rows_reach_their_queries_only(dt, D, Hq, Hkv, T):
    """A row held as NaN makes the queries that see it NaN; earlier ones of the same tile,
    other sequences and rows behind the length keep the bits that they have without it."""
    g, t, S = _gen(D), DT[dt], 150
    held = _held(g, t, 2, Hkv, S, D)
    q = _randn(g, 2, Hq, T, D, dtype=t)
    lens = _ints([100, 120])
    clean = cache4.cache_attention(q, *held, lens, need_lse=True)
    step = held[2].clone()
    step[0, 0, 98] = math.nan        # seen by the last two tokens of head 0's group
    step[:, :, 120:] = math.nan      # behind both lengths
    step[0, :, 100:] = math.nan
    o, lse = cache4.cache_attention(q, held[0], held[1], step, lens, need_lse=True)
    bad = torch.zeros(2, Hq, T, dtype=torch.bool, device=DEV)
    bad[0, :Hq // Hkv, T - 2:] = True
    assert o[bad].isnan().all() and lse[bad].isnan().all()
    assert torch.equal(o[~bad], clean[0][~bad]) and torch.equal(lse[~bad], clean[1][~bad])


def test_queries_that_are_not_finite_are_alone():
    for Hq, T in ((4, 1), (8, 1), (8, 4)):
        g = _gen(T)
        held = _held(g, torch.bfloat16, 1, 1, 90, 64)
        q = _randn(g, 1, Hq, T, 64, dtype=torch.bfloat16)
        clean = cache4.cache_attention(q, *held)
        q[0, 1, 0, 3], q[0, 2, 0, 5] = math.nan, math.inf
        o = cache4.cache_attention(q, *held)
        bad = torch.zeros(1, Hq, T, dtype=torch.bool, device=DEV)
        bad[0, 1, 0] = bad[0, 2, 0] = True
        assert o[bad].isnan().all() and torch.equal(o[~bad], clean[~bad])


def test_the_same_rows_attended_both_ways():
    """Attention over the cache and over the rows read back: the formula's bounds for each, and near each other."""
    g = _gen(11)
    k, v = (_randn(g, 2, 2, 500, 128, dtype=torch.bfloat16) for _ in range(2))
    held = cache4.empty(2, 2, 500, 128)
    cache4.append(*held, k, v, _ints([0, 0]))
    q = _randn(g, 2, 8, 1, 128, dtype=torch.bfloat16)
    lens = _ints([500, 77])
    a, la = cache4.cache_attention(q, *held, lens, need_lse=True)
    b, lb = cache.cache_attention(q, *cache4.read(*held, None, 500), lens, need_lse=True)
    ref.check_attend((a, la), held, q, [500, 77])
    ref.check_attend((b, lb), held, q, [500, 77])


@pytest.mark.parametrize("dt", list(DT))
def test_a_cache_as_it_is_used(dt):
    """A padded prompt, then steps of several tokens and of one, all against 64 bits."""
    g, t, B, Hq, Hkv, D = _gen(7), DT[dt], 3, 8, 2, 64
    c = cache4.KVCache4(B, Hkv, 200, D, dtype=t)
    ks, vs = [[] for _ in range(B)], [[] for _ in range(B)]
    for T, count in ((90, [90, 41, 1]), (5, [5, 2, 0]), (1, None), (1, None), (70, [3, 70, 9])):
        k, v, q = (_randn(g, B, h, T, D, dtype=t) for h in (Hkv, Hkv, Hq))
        c.append(k, v, count=_ints(count))
        o = c.attend(q, count=_ints(count), need_lse=True)
        for b in range(B):
            n = T if count is None else count[b]
            ks[b].append(k[b, :, :n])
            vs[b].append(v[b, :, :n])
        lens = [sum(x.shape[1] for x in y) for y in ks]
        assert c.lens.tolist() == lens
        want = [ref.held(torch.cat(x, 1), torch.cat(y, 1)) for x, y in zip(ks, vs)]
        back = c.read(200, count=c.lens)
        for b in range(B):
            assert all(torch.equal(x[b, :, :lens[b]].cpu().double(), y) for x, y in zip(back, want[b]))
            assert all((x[b, :, lens[b]:] == 0).all() for x in back)
        ref.check_attend(o, (c.k4, c.v4, c.step), q, lens, count)


# ---- calls ---------------------------------------------------------------------
def test_results_repeat_bit_for_bit():
    for Hq, T, S in ((2, 1, 30000), (16, 1, 9000), (16, 40, 3000)):
        g = _gen(T)
        held = _held(g, torch.bfloat16, 2, 2, S, 64)
        q = _randn(g, 2, Hq, T, 64, dtype=torch.bfloat16)
        a = cache4.cache_attention(q, *held, need_lse=True)
        for _ in range(3):
            b = cache4.cache_attention(q, *held, need_lse=True)
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_steps_follow_their_buffers():
    g, B, Hq, Hkv, S, D = _gen(5), 3, 8, 2, 400, 64
    held = _held(g, torch.bfloat16, B, Hkv, S, D)
    q, nk, nv = (_randn(g, B, h, 1, D, dtype=torch.bfloat16) for h in (Hq, Hkv, Hkv))
    q2 = _randn(g, B, Hq, 30, D, dtype=torch.bfloat16)
    lens, start = _ints([1, 200, 400]), _ints([0, 199, 399])

    def step():
        cache4.append(*held, nk, nv, start)
        return (*cache4.cache_attention(q, *held, lens, need_lse=True), cache4.cache_attention(q2, *held, lens),
                *cache4.read(*held, start, 3))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i, n in enumerate(([5, 70, 400], [1, 2, 3], [400, 399, 101], [30, 100, 250])):
        q.copy_(_randn(g, B, Hq, 1, D))
        nk.copy_(_randn(g, B, Hkv, 1, D))
        lens.copy_(_ints(n))
        start.copy_(lens - 1)
        graph.replay()
        a = [x.clone() for x in (*got, *held)]
        torch.cuda.synchronize()
        b = [*step(), *held]
        assert all(torch.equal(x, y) for x, y in zip(a, b)), f"replay {i}"


def test_two_threads_on_their_own_streams(monkeypatch):
    monkeypatch.setattr(cache, "_PLANS_MAX", 3)
    jobs = []
    for i, (Hq, T, S) in enumerate([(2, 1, 700), (8, 30, 500), (16, 1, 4000), (2, 7, 300), (2, 1, 40000), (8, 200, 260)]):
        g = _gen(i)
        held = _held(g, torch.bfloat16, 2, 2, S, 64)
        jobs.append((held, _randn(g, 2, Hq, T, 64, dtype=torch.bfloat16), _randn(g, 2, 2, 40, 64, dtype=torch.bfloat16), _ints([S, S // 2])))

    def run(job):
        held, q, k, lens = job
        mine = [x.clone() for x in held]
        cache4.append(*mine, k, k, _ints([3, 90]))
        return (*cache4.cache_attention(q, *mine, lens, need_lse=True), *cache4.read(*mine, None, 130), *mine)
    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(mine):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    for i in mine:
                        got[i] = run(jobs[i])
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(m,)) for m in ((0, 2, 4), (5, 3, 1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i, w in enumerate(want):
        assert all(torch.equal(a, b) for a, b in zip(w, got[i])), f"job {i}"


def test_what_a_call_writes_counts_as_modified():
    def saved(t):
        return (torch.ones_like(t, requires_grad=True) * t).sum()
    g = _gen(0)
    held = _held(g, torch.bfloat16, 1, 2, 40, 64)
    k = _randn(g, 1, 2, 3, 64, dtype=torch.bfloat16)
    loss = saved(held[2])
    cache4.append(*held, k, k, _ints([3]))
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    out = [torch.zeros(1, 2, 5, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    losses = [saved(x) for x in out]
    cache4.read(*held, None, 5, out=out)
    for x in losses:
        with pytest.raises(RuntimeError, match="inplace operation"):
            x.backward()


def test_empty_calls():
    held = cache4.empty(2, 2, 30, 64)
    q = torch.zeros(2, 4, 0, 64, dtype=torch.bfloat16, device=DEV)
    o, lse = cache4.cache_attention(q, *held, need_lse=True)
    assert o.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)
    cache4.append(*held, q[:, :2], q[:, :2], _ints([0, 0]))
    k, v = cache4.read(*held, None, 0)
    assert k.shape == v.shape == (2, 2, 0, 64)
    # (a fresh cache reads as zeros, and its queries average them)
    q = torch.ones(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV)
    o, lse = cache4.cache_attention(q, *held, need_lse=True)
    assert (o == 0).all() and np.allclose(lse.cpu(), math.log(30), atol=1e-6)


def test_refusals_on_the_gpu():
    held = cache4.empty(2, 2, 64, 64)
    k4, v4, step = held
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV)
    x = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16, device=DEV)
    lens = _ints([64, 64])
    half = cache4.empty(2, 2, 64, 64, dtype=torch.float16)[2]
    bad = [
        (lambda: cache4.cache_attention(q, k4.to(torch.int8), v4, step, lens), "k4 must be"),
        (lambda: cache4.cache_attention(q, k4, v4[:, :, :63], step, lens), "v4 must be"),
        (lambda: cache4.cache_attention(q, k4, v4, step[:, :, :63], lens), "step must be"),
        (lambda: cache4.cache_attention(q, k4, v4, half, lens), "step must be"),
        (lambda: cache4.cache_attention(q.half(), k4, v4, step, lens), "step must be"),
        (lambda: cache4.cache_attention(q, k4, v4, step.transpose(1, 2).contiguous().transpose(1, 2), lens), "steps must be contiguous"),
        (lambda: cache4.cache_attention(q[..., :32], k4, v4, step, lens), "does not go"),
        (lambda: cache4.cache_attention(q[:1], k4, v4, step, lens), "does not go"),
        (lambda: cache4.cache_attention(q[0], k4, v4, step, lens), "4-D"),
        (lambda: cache4.cache_attention(q, k4[0], v4, step, lens), "4-D"),
        (lambda: cache4.cache_attention(q[:, :3], k4, v4, step, lens), "multiple"),
        (lambda: cache4.cache_attention(q, k4[..., 8:24], v4[..., 8:24], step, lens), "does not go|aligned"),
        (lambda: cache4.cache_attention(q[..., :32], k4[..., 8:24], v4[..., 8:24], step, lens), "aligned"),
        (lambda: cache4.cache_attention(q, k4, v4, step, lens[:1]), "lens"),
        (lambda: cache4.cache_attention(q, k4, v4, step, lens.float()), "lens"),
        (lambda: cache4.cache_attention(q, k4, v4, step, lens, count=_ints([1])), "count"),
        (lambda: cache4.cache_attention(q, k4, v4, step, lens, out_gate=q.float()), "out_gate"),
        (lambda: cache4.cache_attention(q, k4, v4, step, lens, scale=math.inf), "scale"),
        (lambda: cache4.cache_attention(q.double(), k4, v4, step, lens), "dtype"),
        (lambda: cache4.cache_attention(q, k4, v4, step, lens.cpu()), "GPU"),
        (lambda: cache4.append(*held, x.float(), x, lens), "v must be"),
        (lambda: cache4.append(*held, x, x[:, :, :2], lens), "v must be"),
        (lambda: cache4.append(*held, x.half(), x.half(), lens), "step must be"),
        (lambda: cache4.append(k4[:1].expand(2, 2, 64, 32), v4, step, x, x, lens), "overlap"),
        (lambda: cache4.append(k4, v4, step[:1].expand(2, 2, 64, 2, 1), x, x, lens), "overlap"),
        (lambda: cache4.append(k4, k4, step, x, x, lens), "same buffer"),
        (lambda: cache4.append(k4, v4, step, k4.view(torch.bfloat16).view(2, 2, -1, 64)[:, :, :3], x, lens), "reads"),
        (lambda: cache4.read(*held, lens, 3, dtype=torch.float16), "step must be"),
        (lambda: cache4.read(*held, lens[:1], 3), "first"),
        (lambda: cache4.read(*held, lens, 4, out=(x, x.clone())), "k must be"),
        (lambda: cache4.read(*held, lens, 3, out=(x, x)), "same buffer"),
        (lambda: cache4.read(*held, lens, 3, out=(x, x[:1].expand(2, 2, 3, 64))), "overlap"),
        (lambda: cache4.read(*held, lens, 3, out=(x, k4.view(torch.bfloat16).view(2, 2, -1, 64)[:, :, :3])), "reads"),
        (lambda: cache4.read(*held, lens, 3, out=(x, x.transpose(2, 3).contiguous().transpose(2, 3))), "contiguous rows"),
    ]
    for i, (call, text) in enumerate(bad):
        with pytest.raises(ValueError, match=text):
            call()
            raise AssertionError(f"call {i} was accepted")


def test_strided_and_misaligned_inputs_are_taken():
    """Queries, gates and new rows in layouts that the kernels do not read are copied."""
    g, held = _gen(2), None
    held = _held(g, torch.bfloat16, 2, 2, 90, 64)
    wide = _randn(g, 2, 4, 2, 72, dtype=torch.bfloat16)
    for q in (wide[..., 4:68], _randn(g, 2, 4, 64, 2, dtype=torch.bfloat16).transpose(2, 3), wide[..., 1:65]):
        a = cache4.cache_attention(q, *held, _ints([90, 3]), out_gate=q)
        assert torch.equal(a, cache4.cache_attention(q.contiguous(), *held, _ints([90, 3]), out_gate=q.contiguous()))
    for k in (wide[:, :2, :, 4:68], _randn(g, 2, 2, 64, 2, dtype=torch.bfloat16).transpose(2, 3)):
        two = [[x.clone() for x in held] for _ in range(2)]
        cache4.append(*two[0], k, k, _ints([5, 6]))
        cache4.append(*two[1], k.contiguous(), k.contiguous(), _ints([5, 6]))
        assert all(torch.equal(x, y) for x, y in zip(*two))
