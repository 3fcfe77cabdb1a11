"""Attention over a cache in 4 bits by tiles of many rows that are not cut, over long
caches: one sequence's many tiles, and more tiles than the card takes several times.
The call's workspace, 256 bytes, says that no tile has parts."""
import pytest
import torch

import _cache4ref as ref
from fbsa_amd import cache, cache4

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _attend(dt, B, Hq, Hkv, T, S, D, lens, count, gated):
    g = torch.Generator(device=DEV).manual_seed(D + B)
    dt = DT[dt]
    k4, v4 = (torch.randint(0, 256, (B, Hkv, S, D // 2), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2))
    step = (0.2 + 0.3 * torch.rand(B, Hkv, S, 2, -(-D // 64), generator=g, device=DEV)).mul(64).round().div(64).to(ref.step_type(dt))
    q, gate = (torch.randn(B, T, Hq, D, generator=g, device=DEV).to(dt).transpose(1, 2) for _ in range(2))
    gate = gate if gated else None
    ints = [None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, count)]
    cache._plans.clear()
    got = cache4.cache_attention(q, k4, v4, step, ints[0], count=ints[1], out_gate=gate, need_lse=True)
    plan, = cache._plans.values()
    assert plan.nbytes == 256
    ref.check_attend(got, (k4, v4, step), q, lens, count, None, gate)


@pytest.mark.parametrize("dt,Hq,Hkv,T,S,D", [("bf16", 128, 128, 600, 1000, 64), ("fp16", 64, 64, 600, 1200, 128), ("bf16", 128, 64, 150, 1500, 256),
                                             ("fp32", 128, 128, 300, 900, 64), ("fp32", 64, 64, 150, 1100, 224), ("fp16", 128, 128, 600, 900, 32)])
@pytest.mark.parametrize("kind", ["behind", "padded", "alone"])
def test_one_sequence(dt, Hq, Hkv, T, S, D, kind):
    """Behind earlier rows, in a padded batch of one, and a prompt that attends itself alone, whose
    tiles see from few keys to all."""
    lens, count = {"behind": (S - 99, None), "padded": (S - 99, T - 23), "alone": (T, None)}[kind]
    _attend(dt, 1, Hq, Hkv, T, S, D, [lens], None if count is None else [count], gated=kind == "padded")


@pytest.mark.parametrize("dt,B,T,S,D", [("bf16", 32, 130, 300, 64), ("fp16", 24, 130, 380, 256), ("fp32", 22, 130, 257, 96), ("fp16", 32, 200, 290, 32)])
def test_many_sequences(dt, B, T, S, D):
    """64 heads of many sequences, of all lengths, some shorter than their new tokens or without any."""
    lens = [S] + [(37 * b * b) % (S + 1) for b in range(1, B)]
    count = [T if b % 3 else (b * 11) % (T + 1) for b in range(B)]
    _attend(dt, B, 64, 64, T, S, D, lens, count, gated=dt != "fp32")
