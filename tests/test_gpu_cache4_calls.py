"""Calls of the 4-bit cache's operators at their limits and in the company they are used in."""
import pytest
import torch

import _cache4ref as ref
from fbsa_amd import cache4

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_more_than_2_26_rows_in_a_call():
    """32 sequences of 8 heads and 262147 rows: 2^26 and some rows written in one call and read in one."""
    B, H, T, D = 32, 8, (1 << 18) + 3, 32
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randn(1, 1, T, D, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    held = cache4.empty(B, H, T, D)
    cache4.append(*held, k.expand(B, H, T, D), v.expand(B, H, T, D), torch.zeros(B, dtype=torch.int32, device=DEV))
    back = cache4.read(*held, None, T)
    for x, want in zip(back, ref.held(k[..., -500:, :], v[..., -500:, :])):
        assert torch.equal(x[B - 1, H - 1, -500:].cpu().double(), want[0, 0])
        assert (x == x[0, 0]).all()
