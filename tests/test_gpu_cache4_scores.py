"""Attention over a cache in 4 bits where scores are infinite: every path, against the formula."""
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
