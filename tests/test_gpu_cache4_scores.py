"""Attention over a cache in 4 bits where scores are infinite or very large: every path, against the formula."""
import math

import pytest
import torch

import _cache4ref as ref
from fbsa_amd import cache4

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
