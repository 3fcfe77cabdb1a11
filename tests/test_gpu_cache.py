"""Cache operators on the GPU against their plain 64-bit forms: lengths of zero
and one and those around a tile, padded batches, rows of NaN behind a sequence,
strided and far-apart caches, every type, head dims that are no power of two."""
import math
import threading

import pytest
import torch

import _cacheref as ref
from fbsa_amd import cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)


def _make(dt, B, Hq, Hkv, T, S, D, lens, seed=0, P=0, layout="bhsd"):
    """Inputs; rows of the caches past each length are NaN."""
    g, dt = _gen(seed), DT[dt]
    q = _randn(g, B, T, Hq, D, dtype=dt).transpose(1, 2)
    if layout == "bhsd":
        k, v = (_randn(g, B, Hkv, S, D, dtype=dt) for _ in range(2))
    elif layout == "bshd":
        k, v = (_randn(g, B, S, Hkv, D, dtype=dt).transpose(1, 2) for _ in range(2))
    else:  # keys and values of a row side by side, with room between rows
        kv = _randn(g, B, Hkv, S, 2, D + 8, dtype=dt)
        k, v = kv[..., 0, :D], kv[..., 1, 8:]
    for b, n in enumerate(lens):
        k[b, :, max(0, n):] = math.nan
        v[b, :, max(0, n):] = math.nan
    kp, vp = (_randn(g, Hkv, P, D, dtype=dt) for _ in range(2)) if P else (None, None)
    return q, k, v, kp, vp, g


def _run(dt, B, Hq, Hkv, T, S, D, lens, count=None, P=0, gate=False, weight=True, scale=None, layout="bhsd", seed=0):
    q, k, v, kp, vp, g = _make(dt, B, Hq, Hkv, T, S, D, lens, seed, P, layout)
    og = _randn(g, B, T, Hq, D, dtype=q.dtype).transpose(1, 2) if gate else None
    w = _randn(g, B, Hkv, S).abs() if weight else None
    out_w = torch.full_like(w, -7.0) if weight else None
    kw = dict(count=_ints(count), scale=scale, out_gate=og, weight=w, out_weight=out_w, need_lse=True)
    if P:
        o, lse = cache.shared_prefix_attention(q, kp, vp, k, v, _ints(lens), **kw)
    else:
        o, lse = cache.cache_attention(q, k, v, _ints(lens), **kw)
    ok = ref.attend(q, k, v, lens, count, kp, vp, scale, og, w)
    if weight:
        for b, n in enumerate(lens):
            n = min(max(n, 0), S)
            assert (out_w[b, :, n:] == -7.0).all(), "rows behind the sequence were written"
            out_w[b, :, n:] = w[b, :, n:]
    both = torch.cat([v.flatten(), vp.flatten()]) if P else v
    ref.check_attend((o, lse, out_w), ok, q, both, S + P, ref.many_rows(q, Hkv, P))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,T", [(4, 4, 1), (8, 2, 1), (16, 1, 5), (3, 1, 40)])
def test_lengths_around_a_tile(dt, D, Hq, Hkv, T):
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 64, 65, 199, 200]
    _run(dt, len(lens), Hq, Hkv, T, 200, D, lens)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [8, 24, 40, 80, 96, 136, 248])
def test_head_dims_between(dt, D):
    _run(dt, 2, 6, 2, 3, 77, D, [77, 50], P=45, gate=True)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [8, 40, 96, 200])
def test_head_dims_between_with_many_rows(dt, D):
    _run(dt, 2, 6, 2, 30, 177, D, [177, 50], P=45, gate=True)
    _run(dt, 1, 5, 1, 61, 300, D, [299], count=[55])


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("P", [1, 31, 32, 33, 500])
@pytest.mark.parametrize("T", [1, 7])
def test_shared_prefix(dt, P, T):
    _run(dt, 5, 8, 2, T, 70, 64, [0, 1, 70, 33, 32], P=P, gate=True)


@pytest.mark.parametrize("P", [0, 129])
def test_padded_batch(P):
    _run("bf16", 6, 4, 2, 9, 300, 128, [300, 9, 5, 1, 0, 120], count=[9, 4, 5, 1, 0, 0], P=P, gate=True)


def test_counts_and_lengths_out_of_range_are_clamped():
    _run("fp16", 4, 4, 4, 3, 64, 64, [-5, 1000, 64, 2], count=[3, 99, -1, 3])


@pytest.mark.parametrize("layout", ["bshd", "packed"])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_layouts(layout, dt):
    _run(dt, 3, 8, 2, 2, 150, 64, [150, 77, 3], layout=layout, P=0, gate=True)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_scales(scale):
    _run("fp32", 2, 2, 1, 2, 90, 32, [90, 41], scale=scale)
    _run("bf16", 2, 4, 1, 2, 90, 64, [90, 41], scale=scale, P=20)
    _run("fp16", 2, 4, 2, 40, 290, 64, [290, 141], scale=scale)


@pytest.mark.parametrize("T,S,lens", [(1, 5000, [5000, 4097]), (70, 1030, [1030, 700]), (257, 600, [600, 258])])
@pytest.mark.parametrize("D", [64, 256])
def test_many_rows_and_shares(T, S, lens, D):
    _run("bf16", 2, 8, 2, T, S, D, lens, count=[T, max(1, T - 3)])


@pytest.mark.parametrize("Hq,Hkv,T,count", [(7, 1, 33, None), (64, 1, 9, [9, 2]), (65, 1, 5, [3, 5]), (96, 1, 3, None), (1, 1, 300, [300, 70])])
def test_weights_of_groups_that_divide_nothing(Hq, Hkv, T, count):
    _run("bf16", 2, Hq, Hkv, T, 400, 32, [400, 290], count=count)


def test_weights_of_queries_before_the_cache():
    # more new tokens than rows: the first ones stand before row 0 and see nothing
    _run("bf16", 3, 8, 2, 50, 140, 64, [20, 140, 1], count=[50, 50, 30])
    _run("bf16", 3, 8, 2, 50, 140, 64, [20, 140, 0], count=[50, 50, 30], P=70)


def test_stacked_prefix_rows():
    _run("bf16", 37, 8, 2, 2, 40, 128, [3 + b for b in range(37)], P=1000)


@pytest.mark.parametrize("T,P", [(2, 0), (40, 0), (2, 50), (40, 300)])
def test_padding_may_hold_anything(T, P):
    """Queries and gates past a sequence's count, and rows past its length, are NaN."""
    count, lens = [T, T // 2, 0], [T + 60, T // 2, 9]
    q, k, v, kp, vp, g = _make("bf16", 3, 8, 2, T, T + 60, 64, lens, P=P)
    og, w = _randn(g, 3, 8, T, 64, dtype=q.dtype), _randn(g, 3, 2, T + 60).abs()
    bad = [x.clone() for x in (q, og)]
    for b, c in enumerate(count):
        for x in bad:
            x[b, :, c:] = math.nan
    a, b = torch.zeros_like(w), torch.zeros_like(w)

    def call(q, og, out):
        kw = dict(count=_ints(count), out_gate=og, weight=w, out_weight=out, need_lse=True)
        return (cache.shared_prefix_attention(q, kp, vp, k, v, _ints(lens), **kw) if P else
                cache.cache_attention(q, k, v, _ints(lens), **kw))
    want, got = call(q, og, a), call(*bad, b)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1]) and torch.equal(a, b)
    assert (got[0][2] == 0).all() and not torch.isnan(b).any()


def test_weight_in_place_from_nothing_and_absent():
    q, k, v, _, _, g = _make("bf16", 2, 4, 2, 1, 100, 64, [100, 60])
    lens, w = _ints([100, 60]), _randn(g, 2, 2, 100).abs()
    a = torch.full_like(w, 3.0)
    o1 = cache.cache_attention(q, k, v, lens, weight=w, out_weight=a)
    before = w.clone()
    o2 = cache.cache_attention(q, k, v, lens, weight=w)
    assert torch.equal(o1, o2)
    assert torch.equal(w[0], a[0]) and torch.equal(w[1, :, :60], a[1, :, :60]) and torch.equal(w[1, :, 60:], before[1, :, 60:])
    c = torch.full_like(w, 5.0)
    o3 = cache.cache_attention(q, k, v, lens, out_weight=c)
    assert torch.equal(o1, o3) and torch.equal(o1, cache.cache_attention(q, k, v, lens))
    # one query per head gives a total of one
    assert (c[0].sum(-1) - 2).abs().max() < 200 * 2.0 ** -24 and (c[1, :, 60:] == 5.0).all()


def test_no_lengths_is_the_capacity_and_int64_lengths():
    q, k, v, _, _, _ = _make("fp16", 2, 4, 4, 2, 50, 64, [50, 50])
    a = cache.cache_attention(q, k, v)
    assert torch.equal(a, cache.cache_attention(q, k, v, torch.tensor([50, 50], device=DEV)))


def test_far_rows_and_sequences():
    # rows 32 MiB apart and sequences past 2^32 bytes: every offset has 64 bits
    g, B, S, D = _gen(3), 2, 140, 64
    big = torch.empty(B * S * (1 << 24), dtype=torch.bfloat16, device=DEV)
    k = big.as_strided((B, 1, S, D), (S * (1 << 24), 0, 1 << 24, 1))
    v = big.as_strided((B, 1, S, D), (S * (1 << 24), 0, 1 << 24, 1), 4096)
    k.copy_(_randn(g, B, 1, S, D))
    v.copy_(_randn(g, B, 1, S, D))
    q, w = _randn(g, B, 2, 1, D, dtype=torch.bfloat16), torch.zeros(B, 1, S, device=DEV)
    near = [x.contiguous() for x in (k, v)]
    lens = _ints([140, 133])
    o = cache.cache_attention(q, k, v, lens, weight=w)
    assert torch.equal(o, cache.cache_attention(q, *near, lens))
    # many rows, and far-apart queries, prefixes and outputs of an eviction
    q = torch.empty(B * 2 * 40 * (1 << 23), dtype=torch.bfloat16, device=DEV).as_strided(
        (B, 2, 40, D), (2 * 40 * (1 << 23), 40 * (1 << 23), 1 << 23, 1)).copy_(_randn(g, B, 2, 40, D))
    a, b = torch.zeros_like(w), torch.zeros_like(w)
    o = cache.shared_prefix_attention(q, k[1], v[1], k, v, lens, out_weight=a)
    assert torch.equal(o, cache.shared_prefix_attention(q.contiguous(), near[0][1], near[1][1], *near, lens, out_weight=b))
    assert torch.equal(a, b)
    wide = (big.as_strided((B, 1, 70, D), (S * (1 << 24), 0, 1 << 24, 1), 8192), big.as_strided(
        (B, 1, 70, D), (S * (1 << 24), 0, 1 << 24, 1), 12288), torch.zeros(B, 1, 70, device=DEV))
    with pytest.raises(ValueError, match="overlaps"):
        cache.evict(k, v, w, lens, 70, out=wide)  # (interleaved rows of one buffer: told apart by their span only)
    thin = tuple(x.contiguous() for x in wide)
    assert torch.equal(cache.evict(k, v, w, lens, 70, out=thin)[0], cache.evict(*near, w, lens, 70, out=thin)[0])
    new = [_randn(g, B, 1, 3, D, dtype=torch.bfloat16) for _ in range(2)]
    for caches in ((k, v), near):
        cache.append(*caches, *new, _ints([136, 130]))
    assert torch.equal(k, near[0]) and torch.equal(v, near[1])
    w2 = w.clone()
    index, n = cache.evict(k, v, w, lens, 70, recent=4)
    index2, _ = cache.evict(*near, w2, lens, 70, recent=4)
    assert torch.equal(index, index2) and torch.equal(k, near[0]) and torch.equal(v, near[1]) and torch.equal(w, w2)


def test_repeats_and_streams_are_bitwise_equal():
    q, k, v, kp, vp, g = _make("bf16", 4, 16, 2, 1, 900, 128, [900, 13, 500, 0], P=700)
    lens, w = _ints([900, 13, 500, 0]), torch.zeros(4, 2, 900, device=DEV)

    def call():
        out = torch.zeros_like(w)
        return [*cache.shared_prefix_attention(q, kp, vp, k, v, lens, out_weight=out, need_lse=True), out]
    a = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = call()
    c = call()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [8, 64, 200])
def test_append(dt, D):
    g, dt, B, H, S, T = _gen(1), DT[dt], 7, 3, 50, 6
    k, v = _randn(g, B, H, S, D, dtype=dt), _randn(g, B, S, H, D, dtype=dt).transpose(1, 2)
    new = [_randn(g, B, T, H, D, dtype=dt).transpose(1, 2) for _ in range(2)]
    w = _randn(g, B, H, S)
    start, count = [0, 44, 47, 50, -2, 10, -(2 ** 31)], [6, 6, 6, 6, 6, 0, 99]
    want = [x.clone() for x in (k, v, w)]
    for b in range(B):
        for t in range(min(T, count[b])):
            if 0 <= start[b] + t < S:
                want[0][b, :, start[b] + t], want[1][b, :, start[b] + t] = new[0][b, :, t], new[1][b, :, t]
                want[2][b, :, start[b] + t] = 0
    cache.append(k, v, *new, _ints(start), count=_ints(count), weight=w)
    assert all(torch.equal(x, y) for x, y in zip((k, v, w), want))
    cache.append(k, v, new[0][:, :, :0], new[1][:, :, :0], _ints(start))  # nothing to write
    odd = torch.empty(B, H, T, D + 1, dtype=dt, device=DEV)[..., 1:]      # rows off 16 bytes: copied first
    odd.copy_(new[0])
    cache.append(k, v, odd, odd, torch.zeros(B, dtype=torch.int64, device=DEV))
    assert torch.equal(k[:, :, :T], odd) and torch.equal(v[:, :, :T], odd)


def _evict_case(dt, B, H, S, D, lens, budget, recent, sink, kind, inplace, seed=0):
    g, dt = _gen(seed), DT[dt]
    k, v = (_randn(g, B, H, S, D, dtype=dt) for _ in range(2))
    w = _randn(g, B, H, S)
    if kind == "ties":
        w = (w * 2).round()
    elif kind == "equal":
        w.fill_(0.25)
    elif kind == "odd":
        u = torch.rand(B, H, S, generator=g, device=DEV)
        for x, lo in ((math.nan, 0.1), (math.inf, 0.2), (-math.inf, 0.3), (0.0, 0.5), (-0.0, 0.7)):
            w = w.masked_fill((u < lo) & (u >= lo - 0.1), x)
    keep = ref.evict(k, v, w.cpu(), lens, budget, recent, sink)
    before = [x.clone() for x in (k, v, w)]
    if inplace:
        out = (k, v, w)
        index, n = cache.evict(k, v, w, _ints(lens), budget, recent=recent, sink=sink)
        old = before
    else:
        SO = min(budget, S) + 3
        out = (_randn(g, B, SO, H, D, dtype=dt).transpose(1, 2), _randn(g, B, H, SO, D, dtype=dt), _randn(g, B, H, SO))
        old = [x.clone() for x in out]
        index, n = cache.evict(k, v, w, _ints(lens), budget, recent=recent, sink=sink, out=out)
        assert all(torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0)) for x, y in zip((k, v, w), before))
    assert index.shape == (B, H, min(budget, S))
    for b in range(B):
        for h in range(H):
            rows = keep[b * H + h]
            assert int(n[b]) == len(rows)
            assert index[b, h].tolist() == rows + [-1] * (index.shape[2] - len(rows))
            for x, src, was in zip(out, before, old):
                want = was[b, h].clone()
                want[:len(rows)] = src[b, h, rows]
                assert torch.equal(x[b, h].nan_to_num(9.0), want.nan_to_num(9.0))


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd"])
@pytest.mark.parametrize("budget,recent,sink", [(1, 0, 0), (64, 10, 4), (64, 60, 4), (1500, 0, 0), (1999, 100, 1), (5000, 7, 7)])
def test_evict(inplace, kind, budget, recent, sink):
    _evict_case("bf16", 6, 2, 2500, 64, [2500, 0, 1, 64, 65, 2047], budget, recent, sink, kind, inplace)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("dt,D", [("fp32", 256), ("fp16", 8), ("bf16", 200)])
def test_evict_types_and_widths(inplace, dt, D):
    _evict_case(dt, 2, 3, 1300, D, [1300, 1025], 1024, 128, 4, "ties", inplace)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd"])
@pytest.mark.parametrize("budget,recent,sink", [(20000, 512, 4), (9000, 8500, 500), (69999, 0, 0), (8, 0, 8)])
def test_evict_long(inplace, kind, budget, recent, sink):
    _evict_case("bf16", 3, 2, 70001, 16, [70001, 33000, 8192], budget, recent, sink, kind, inplace)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("S", [2048, 8192, 16384, 32768])
def test_evict_at_each_register_count(inplace, S):
    _evict_case("fp16", 2, 1, S, 16, [S, S - 1], S // 3, 100, 4, "ties", inplace)


@pytest.mark.parametrize("kind", ["random", "ties", "equal"])
def test_evict_of_very_long_sequences(kind):
    # more chunks of a sequence than are ranked at a time (64 of 8192 rows)
    _evict_case("bf16", 2, 1, 560000, 8, [560000, 524289], 30000, 600, 4, kind, False)


def test_evict_again():
    # rows that were kept before lie in the first places and outweigh the rest
    g, B, H, S, D, budget = _gen(7), 1, 2, 40000, 16, 6000
    k, v = (_randn(g, B, H, S, D, dtype=torch.bfloat16) for _ in range(2))
    w = torch.rand(B, H, S, generator=g, device=DEV)
    w[:, :, :budget] += 0.5
    w[:, :, :2048] = 0.75
    before = [x.clone() for x in (k, v, w)]
    keep = ref.evict(k, v, w.cpu(), [S], budget, 100, 4)
    index, _ = cache.evict(k, v, w, _ints([S]), budget, recent=100, sink=4)
    for h in range(H):
        assert index[0, h].tolist() == keep[h]
        for x, y in zip((k, v, w), before):
            assert torch.equal(x[0, h, :budget], y[0, h, keep[h]]) and torch.equal(x[0, h, budget:], y[0, h, budget:])


def test_evict_in_place_in_parts():
    # more kept rows than pass through the workspace at a time: 8192 of these heads
    _evict_case("bf16", 2, 8, 30000, 64, [30000, 26000], 20001, 300, 4, "random", True)
    _evict_case("bf16", 2, 8, 30000, 64, [20000, 29999], 20001, 300, 4, "equal", True)


@pytest.mark.parametrize("budget", [512, 513, 1100])
def test_evict_in_place_of_strided_caches(budget):
    g, B, H, S, D = _gen(5), 2, 3, 1500, 40
    kv = _randn(g, B, S, 2, H, D, dtype=torch.bfloat16)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    w, lens, before = _randn(g, B, H, S), [S, budget + 1], kv.clone()
    keep = ref.evict(k, v, w.cpu(), lens, budget, 17, 3)
    index, n = cache.evict(k, v, w, _ints(lens), budget, recent=17, sink=3)
    want = before.clone()
    for b in range(B):
        for h in range(H):
            rows = keep[b * H + h]
            assert index[b, h].tolist() == rows and int(n[b]) == budget
            want[b, :budget, :, h] = before[b, rows][:, :, h]
    assert torch.equal(kv, want)


def test_evict_in_place_replayed():
    # a captured call, new rows before every replay, eager calls between them
    g, B, H, S, D, budget = _gen(6), 1, 4, 3000, 64, 2000
    k, v = (torch.zeros(B, H, S, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    w = torch.zeros(B, H, S, device=DEV)
    lens = _ints([S])
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        cache.evict(k, v, w, lens, budget)
    torch.cuda.current_stream().wait_stream(stream)
    with torch.cuda.graph(graph):
        index, n = cache.evict(k, v, w, lens, budget, recent=10)
    for _ in range(4):
        new = [_randn(g, *x.shape, dtype=x.dtype) for x in (k, v, w)]
        eager = [x.clone() for x in new]
        cache.evict(*eager, lens, budget, recent=10)
        for x, y in zip((k, v, w), new):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((k, v, w), eager))


def test_evict_lengths_past_the_capacity():
    _evict_case("bf16", 3, 1, 100, 32, [400, -3, 100], 60, 3, 2, "random", False)


def test_decode_loop():
    """append -> attend -> evict over sequences of different lengths, behind a
    shared prompt, against the same steps in 64 bits on the rows kept so far."""
    g, B, Hq, Hkv, S, D, P, budget = _gen(11), 3, 8, 2, 96, 64, 75, 40
    c = cache.KVCache(B, Hkv, S, D, dtype=torch.bfloat16, weight=True)
    kp, vp = (_randn(g, Hkv, P, D, dtype=torch.bfloat16) for _ in range(2))
    mine = [[torch.zeros(Hkv, 0, D, dtype=torch.bfloat16, device=DEV) for _ in range(B)] for _ in range(2)]
    for step, (T, counts) in enumerate([(50, [50, 20, 1]), (1, None), (1, None), (3, [3, 0, 2]), (30, None), (1, None)]):
        new = [_randn(g, B, T, Hkv, D, dtype=torch.bfloat16).transpose(1, 2) for _ in range(2)]
        q = _randn(g, B, T, Hq, D, dtype=torch.bfloat16).transpose(1, 2)
        count = counts or [T] * B
        w0 = c.weight.clone()
        for b in range(B):
            n = int(c.lens[b])
            w0[b, :, n:n + count[b]] = 0
            for x in range(2):
                mine[x][b] = torch.cat([mine[x][b], new[x][b, :, :count[b]]], 1)
        c.append(*new, count=_ints(counts))
        lens = c.lens.tolist()
        assert lens == [x.shape[1] for x in mine[0]]
        o, lse = c.attend(q, prefix=(kp, vp), count=_ints(counts), need_lse=True)
        dense = [torch.zeros(B, Hkv, S, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        for b in range(B):
            for x in range(2):
                dense[x][b, :, :lens[b]] = mine[x][b]
        want = ref.attend(q, *dense, lens, count, kp, vp, weight=w0)
        ref.check_attend((o, lse, c.weight), want, q, torch.cat([dense[1].flatten(), vp.flatten()]), S + P,
                         ref.many_rows(q, Hkv, P))
        keep = ref.evict(c.k, c.v, c.weight.cpu(), lens, budget, 8, 2)
        index = c.evict(budget, recent=8, sink=2)
        assert c.lens.tolist() == [min(n, budget) for n in lens]
        for b in range(B):
            for x in range(2):
                mine[x][b] = torch.stack([mine[x][b][h, keep[b * Hkv + h]] for h in range(Hkv)])
            for h in range(Hkv):
                assert index[b, h, :c.lens[b]].tolist() == keep[b * Hkv + h]


def test_captured_steps_follow_their_buffers():
    """A captured step replayed with other lengths and inputs in its buffers, the
    program's own work between: every replay against the eager call."""
    g, B, Hq, Hkv, S, D, P = _gen(5), 3, 8, 2, 400, 64, 300
    k, v = (_randn(g, B, Hkv, S, D, dtype=torch.bfloat16) for _ in range(2))
    kp, vp = (_randn(g, Hkv, P, D, dtype=torch.bfloat16) for _ in range(2))
    q, nk, nv = (_randn(g, B, h, 1, D, dtype=torch.bfloat16) for h in (Hq, Hkv, Hkv))
    lens, start = _ints([1, 200, 400]), _ints([0, 199, 399])
    w = _randn(g, B, Hkv, S).abs()
    out_w = torch.zeros_like(w)
    out = (torch.zeros(B, Hkv, 100, D, dtype=torch.bfloat16, device=DEV), torch.zeros(B, Hkv, 100, D, dtype=torch.bfloat16, device=DEV),
           torch.zeros(B, Hkv, 100, device=DEV))

    def step():
        cache.append(k, v, nk, nv, start, weight=w)
        o = cache.shared_prefix_attention(q, kp, vp, k, v, lens, weight=w, out_weight=out_w)
        p = cache.cache_attention(q, k, v, lens)
        index, n = cache.evict(k, v, out_w, lens, 100, recent=10, sink=1, out=out)
        return o, p, index, n
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i, n in enumerate(([5, 70, 400], [1, 2, 3], [400, 399, 101], [0, 100, 250])):
        q.copy_(_randn(g, B, Hq, 1, D))
        nk.copy_(_randn(g, B, Hkv, 1, D))
        lens.copy_(_ints(n))
        start.copy_(lens - 1)
        w.copy_(_randn(g, B, Hkv, S).abs())
        for x in (out_w, *out):
            x.zero_()
        graph.replay()
        a = [x.clone() for x in (*got, out_w, *out, k, v)]
        torch.cuda.synchronize()
        for x in (out_w, *out):
            x.zero_()
        b = [*step(), out_w, *out, k, v]
        assert all(torch.equal(x, y) for x, y in zip(a, b)), f"replay {i}"


def test_two_threads_on_their_own_streams(monkeypatch):
    """Two host threads at once, each on a stream of its own, the plans turned over
    all the while: every result as in sequence."""
    monkeypatch.setattr(cache, "_PLANS_MAX", 3)
    jobs = []
    for i, (T, P, S) in enumerate([(1, 0, 700), (30, 0, 500), (1, 400, 90), (7, 90, 300), (1, 0, 40000), (200, 0, 260)]):
        q, k, v, kp, vp, g = _make("bf16", 2, 8, 2, T, S, 64, [S, S // 2], seed=i, P=P)
        jobs.append((q, k, v, kp, vp, _ints([S, S // 2]), _randn(g, 2, 2, S).abs()))

    def run(job):
        q, k, v, kp, vp, lens, w = job
        out = torch.zeros_like(w)
        o = (cache.cache_attention(q, k, v, lens, weight=w, out_weight=out) if kp is None else
             cache.shared_prefix_attention(q, kp, vp, k, v, lens, weight=w, out_weight=out))
        rows = (torch.zeros_like(k[:, :, :50]), torch.zeros_like(v[:, :, :50]), torch.zeros_like(w[:, :, :50]))
        index, _ = cache.evict(k, v, out, lens, 50, recent=5, out=tuple(x.contiguous() for x in rows))
        return o, out, index
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


def test_refusals_on_the_gpu():
    q, k, v, kp, vp, g = _make("bf16", 2, 4, 2, 1, 64, 64, [64, 64], P=16)
    lens, w = _ints([64, 64]), torch.zeros(2, 2, 64, device=DEV)
    bad = [
        (lambda: cache.cache_attention(q, k.float(), v, lens), "k must be"),
        (lambda: cache.cache_attention(q, k, v[:, :, :63], lens), "v must be"),
        (lambda: cache.cache_attention(q[..., :60], k[..., :60], v[..., :60], lens), "head dim|aligned"),
        (lambda: cache.cache_attention(q, k[..., :56], v[..., :56], lens), "k must be"),
        (lambda: cache.cache_attention(q, k.transpose(2, 3).contiguous().transpose(2, 3), v, lens), "contiguous rows"),
        (lambda: cache.cache_attention(q[:, :3], k, v, lens), "multiple"),
        (lambda: cache.cache_attention(q, k, v, lens[:1]), "lens"),
        (lambda: cache.cache_attention(q, k, v, lens.float()), "lens"),
        (lambda: cache.cache_attention(q, k, v, lens, count=_ints([1])), "count"),
        (lambda: cache.cache_attention(q, k, v, lens, out_gate=q.float()), "out_gate"),
        (lambda: cache.cache_attention(q, k, v, lens, weight=w.double()), "out_weight"),
        (lambda: cache.cache_attention(q, k, v, lens, weight=w, out_weight=w.expand(2, 2, 64)[:, :, 1:]), "out_weight"),
        (lambda: cache.cache_attention(q, k, v, lens, out_weight=w[:1, :1].expand(2, 2, 64)), "overlap"),
        (lambda: cache.cache_attention(q, k, v, lens, scale=math.inf), "scale"),
        (lambda: cache.cache_attention(q.double(), k.double(), v.double(), lens), "dtype"),
        (lambda: cache.cache_attention(q.requires_grad_(), k, v, lens), "gradients"),
        (lambda: cache.shared_prefix_attention(q.detach(), kp, vp[:, :8], k, v, lens), "v_prefix"),
        (lambda: cache.shared_prefix_attention(q.detach(), None, vp, k, v, lens), "required"),
        (lambda: cache.shared_prefix_attention(q.detach(), kp[None], vp[None], k, v, lens), "3-D"),
        (lambda: cache.append(k, v, k[:, :, :2], v[:, :, 62:], lens), "reads"),
        (lambda: cache.append(k, k, kp[None, :, :1].repeat(2, 1, 1, 1), kp[None, :, :1].repeat(2, 1, 1, 1), lens), "same buffer"),
        (lambda: cache.append(k[:1].expand(2, 2, 64, 64), v, q.detach()[:, :2], q.detach()[:, :2], lens), "overlap"),
        (lambda: cache.evict(k, v, w, lens, 0), "positive"),
        (lambda: cache.evict(k, v, w, lens, 8, recent=5, sink=4), "budget"),
        (lambda: cache.evict(k, v, w, lens, 8, out=(k, v, w)), "reads"),
        (lambda: cache.evict(k, v, w, lens, 8, out=(k.clone()[:, :, :7], v.clone()[:, :, :7], w.clone()[:, :, :7])), "capacity"),
        (lambda: cache.KVCache(1, 1, 8, 64).evict(4), "weights"),
    ]
    for i, (call, text) in enumerate(bad):
        with pytest.raises(ValueError, match=text):
            call()
            raise AssertionError(f"call {i} was accepted")
    with torch.no_grad():
        cache.cache_attention(q, k, v, lens)  # q still asks for gradients
    empty = cache.cache_attention(q.detach()[:, :, :0], k, v, lens, need_lse=True)
    assert empty[0].shape == (2, 4, 0, 64) and empty[1].shape == (2, 4, 0)
    same = cache.shared_prefix_attention(q.detach(), kp[:, :0], vp[:, :0], k, v, lens)
    assert torch.equal(same, cache.cache_attention(q.detach(), k, v, lens))
