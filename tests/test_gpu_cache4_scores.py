"""Attention over a cache in 4 bits where scores are infinite, very large or far apart: every path, against the formula."""
import math

import pytest
import torch

import _cache4ref as ref
from fbsa_amd import cache, cache4

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# rows of a KV head: waves with 4, 2 and 1 parts of a chunk, two tiles a wave, 64 and 128 rows a workgroup
ROWS = [(2, 1), (4, 2), (4, 4), (8, 4), (8, 7), (8, 30)]


def _held(seed, dt, S, D):
    """One sequence and KV head of random codes and steps: (k4, v4, step)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    k4, v4 = (torch.randint(0, 256, (1, 1, S, D // 2), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2))
    step = (0.2 + 0.3 * torch.rand(1, 1, S, 2, -(-D // 64), generator=g, device=DEV)).mul(64).round().div(64)
    return k4, v4, step.to(ref.step_type(dt))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("Hq,T", ROWS)
@pytest.mark.parametrize("S", [90, 3000])
def test_infinite_queries(dt, D, Hq, T, S):
    """A query of which one element is infinite scores every key -inf (no weights: 0 and
    -inf), or some key +inf (NaN), as the formula says, in 32 bits as in 16. Queries with
    an infinity against one of its own sign are NaN; finite ones keep their bits."""
    dt = DT[dt]
    k4, v4, step = _held(D + T, dt, S, D)
    # element 6 of every key positive, but negative in the last row
    k4[..., 3] = k4[..., 3] & 0xf0 | 5
    k4[:, :, S - 1, 3] |= 8
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(1, Hq, T, D, generator=g, device=DEV).to(dt)
    clean = cache4.cache_attention(q, k4, v4, step, need_lse=True)
    q[0, 0, :, 6] = -math.inf
    q[0, 1, :, 6] = math.inf
    o, lse = cache4.cache_attention(q, k4, v4, step, need_lse=True)
    # head 0 sees only positive elements before the last token, which sees the last row
    assert (o[0, 0, :T - 1] == 0).all() and (lse[0, 0, :T - 1] == -math.inf).all()
    assert o[0, 0, T - 1].isnan().all() and o[0, 1].isnan().all()
    assert not lse[0, 0, T - 1].isfinite() and not lse[0, 1].isfinite().any()
    assert torch.equal(o[0, 2:], clean[0][0, 2:]) and torch.equal(lse[0, 2:], clean[1][0, 2:])
    # NaN stays NaN, whichever of its bits are set
    if dt == torch.float32:
        q.view(torch.int32)[0, 0, :, 6] = 0x7f800001
        assert cache4.cache_attention(q, k4, v4, step)[0, 0].isnan().all()


def _uniform(dt, S, D, keys, values):
    """One sequence and KV head whose row s is all keys[s], all values[s] (codes' numbers, steps of 1)."""
    code = {0.0: 0, 0.5: 1, 1.0: 2, 1.5: 3, 2.0: 4, 3.0: 5, 4.0: 6, 6.0: 7}

    def codes(x):
        c = torch.tensor([code[abs(y)] + 8 * (y < 0) for y in x], dtype=torch.uint8, device=DEV)
        return (c * 17).view(1, 1, S, 1).expand(1, 1, S, D // 2).contiguous()
    return codes(keys), codes(values), torch.ones(1, 1, S, 2, -(-D // 64), dtype=ref.step_type(dt), device=DEV)


@pytest.mark.parametrize("D,T,H", [(64, 300, 256), (128, 300, 256), (256, 130, 256), (256, 60, 512)])
@pytest.mark.parametrize("first", [True, False])
def test_many_small_probabilities_in_fp16(D, T, H, first):
    """131072 keys 2^-25.3 below one that holds nearly all of a query's weight, in one share:
    their 0.3% arrives (P in fp16 with 7 of its binades below: 0.3% of the row sum and
    none of the result without them). With scale 1 / D and keys of 0 and 1 a query of
    17.53125 has that score. Each p is off by h = 2^-11 of itself or, below 2^-14, by half
    an fp16 step 2^-24 over 2^7, the row sum being at least 1: 2^-32. So o is off by h for P,
    h for its storage, and 2^-32 sum |v|. Sums: a lane's row sum takes a step a chunk of 64
    keys, an element of O two, each off by up to 2^-24 of what is there (the largest key's
    weight, 1, and less than 2^-6 more), and the small terms being equal the roundings can go one way:
    S / 64 2^-24 of the row sum, twice that of o; 2^-20 for the exponentials of either."""
    S, h, a = 131072 + T, 2.0 ** -11, 17.53125
    top = 0 if first else S - T - 1
    keys, values = [0.0] * S, [6.0] * S
    keys[top], values[top] = 1.0, 1.0
    held = [x.expand(1, H, *x.shape[2:]) for x in _uniform(torch.float16, S, D, keys, values)]
    q = torch.full((1, H, T, D), a, dtype=torch.float16, device=DEV)
    o, lse = cache4.cache_attention(q, *held, scale=1.0 / D, need_lse=True)
    assert next(reversed(cache._plans.values())).nbytes == 256   # one share a tile
    seen = torch.arange(S - T + 1, S + 1, dtype=torch.float64).view(1, 1, T, 1)
    w = (seen - 1) * math.exp(-a)
    want = (1 + 6 * w) / (1 + w)
    err = (o.cpu().double() - want).abs()
    steps = (S / 64 + 1) * 2.0 ** -24
    assert (err <= (2 * h + 3 * steps + 2.0 ** -19) * want + 2.0 ** -32 * 6 * seen).all(), f"{float(err.max()):.2e}"
    # (the numbers near 17.5 are 2^-19 apart)
    assert (lse.cpu().double() - (a + w.log1p()).squeeze(-1)).abs().max() <= steps + 2.0 ** -20 + 2.0 ** -19


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("Hq,T", ROWS)
@pytest.mark.parametrize("S", [70, 2000])
def test_scores_of_any_size(dt, D, Hq, T, S):
    """Scores of 2^20 to 2^110, either sign: the largest has all the weight, though neighbouring
    32-bit numbers there are further apart than an exponential reaches. Queries of 1 and
    -1 and keys of whole codes have exact sums; the next score is a quarter of the largest below it."""
    g = torch.Generator().manual_seed(S + T)
    keys = [(1.0, 1.5, 2.0, 3.0)[i] for i in torch.randint(0, 4, (S,), generator=g)]
    values = [(-6.0, -3.0, -1.0, 0.5, 1.5, 4.0)[i] for i in torch.randint(0, 6, (S,), generator=g)]
    for s, x in ((5, 4.0), (6, 0.5), (S - T, 6.0)):
        keys[s] = x
    dt = DT[dt]
    held = _uniform(dt, S, D, keys, values)
    sign = torch.ones(Hq)
    sign[1::2] = -1
    q = sign.view(1, Hq, 1, 1).expand(1, Hq, T, D).to(DEV, dt).contiguous()
    want = torch.tensor([values[S - T] if x > 0 else values[6] for x in sign], dtype=torch.float64)
    for scale in (12345.6789, 2.1e5, 3.1e5, 4.1e6, 3.3e7, 7.7e9, 1.234e13, 5.4321e20, 9.87e30):
        o, lse = cache4.cache_attention(q, *held, scale=scale, need_lse=True)
        off = (o.cpu().double() - want.view(1, Hq, 1, 1)).abs() / want.abs().view(1, Hq, 1, 1)
        assert off.max() <= (2.0 ** -20 if dt == torch.float32 else 0.0), f"scale {scale}"
        score = D * scale * torch.where(sign > 0, 6.0, -0.5).double()
        assert ((lse.cpu().double() - score.view(1, Hq, 1)) / score.view(1, Hq, 1)).abs().max() <= 2.0 ** -21, f"scale {scale}"


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("Hq,T", ROWS)
@pytest.mark.parametrize("S", [200, 3000])
def test_very_large_scores_beside_small_ones(dt, D, Hq, T, S):
    """Scores of 0 and, in some rows, 2^20 to 2^110: where those are positive (even heads) the
    one of them at the end of what all queries see has all the weight, where negative the zeros share it
    and nothing else adds. Their mean: sums of values that are multiples of 0.5, exact in 32 bits but for the
    probabilities' 2^-20 (16-bit ones exact: they are 1), the division and the storage."""
    g = torch.Generator().manual_seed(S + T)
    values = [(-6.0, -3.0, 1.5, 4.0)[i] for i in torch.randint(0, 4, (S,), generator=g)]
    keys = [0.0] * S
    for s in (*range(3, S - T, 71), S - T - 1):
        keys[s] = 4.0
    keys[S - T - 1] = 6.0
    dt = DT[dt]
    held = _uniform(dt, S, D, keys, values)
    sign = torch.ones(Hq)
    sign[1::2] = -1
    q = sign.view(1, Hq, 1, 1).expand(1, Hq, T, D).to(DEV, dt).contiguous()
    zero, v = torch.tensor(keys) == 0, torch.tensor(values, dtype=torch.float64)
    seen = torch.arange(S).view(1, S) <= torch.arange(S - T, S).view(T, 1)
    n = (seen & zero).sum(1)
    mean = ((seen & zero).double() @ v) / n
    h = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    for scale in (12345.6789, 3.1e5, 3.3e7, 5.4321e20, 9.87e30):
        o, lse = (x.cpu().double() for x in cache4.cache_attention(q, *held, scale=scale, need_lse=True))
        for head in range(Hq):
            if head % 2:
                assert ((o[0, head] - mean.view(T, 1)).abs() <= (h + 2.0 ** -18) * mean.abs().view(T, 1) + 2.0 ** -18).all(), f"scale {scale}"
                assert (lse[0, head] - n.double().log()).abs().max() <= 2.0 ** -18, f"scale {scale}"
            else:
                assert (o[0, head] - values[S - T - 1]).abs().max() <= 2.0 ** -18, f"scale {scale}"
                assert (lse[0, head] / (6.0 * D * scale) - 1).abs().max() <= 2.0 ** -21, f"scale {scale}"
