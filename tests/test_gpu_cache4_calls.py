"""Calls of the 4-bit cache's operators at their limits and in the company they are used in."""
import pytest
import torch

import _cache4ref as ref
import _cachetight as tight
from _util import assert_close, np64
from fbsa_amd import _lib, cache4, ops
from oracle import attn as oattn, select as osel

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


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 160])
def test_how_far_off_an_element_is(dt, D):
    """An element is off by (1 + 2^-6) / 6 of its group's largest magnitude at most: codes are two
    steps apart at the widest, and a step of 6 significant bits is up to 2^-6 above a sixth of
    the largest. It is off by more than a sixth, too. Steps have a last bit of at least 2^-125, fp16's 2^-23:
    half of that more in a step, so up to 6 halves in an element."""
    least = 2.0 ** (-24 if dt == torch.float16 else -126)
    g = torch.Generator(device=DEV).manual_seed(D)
    x = torch.randn(1, 2, 4000, D, generator=g, device=DEV)
    x *= torch.exp2(torch.randint(-20, 14, (1, 2, 4000, 1), generator=g, device=DEV).float())
    x[0, 0, 0, :2] = torch.tensor([6.125, 5.15625])
    x[0, 0, 0, 2:] = 0
    x[0, 0, 1] = 2.0 ** -22   # (fp16: a sixth is below half of the least step, so zeros)
    x = x.to(dt)
    held = cache4.empty(1, 2, 4000, D, dtype=dt)
    cache4.append(*held, x, x, torch.zeros(1, dtype=torch.int32, device=DEV))
    back = cache4.read(*held, None, 4000, dtype=dt)[0].double()
    x = x.double()
    off = (back - x).abs()
    for i in range(0, D, 64):
        most = x[..., i:i + 64].abs().amax(-1, keepdim=True)
        assert (off[..., i:i + 64] <= (1 + 2.0 ** -6) / 6 * most + 6 * least).all()
    assert off[0, 0, 0, 1] > x[0, 0, 0, 0] / 6
    if dt == torch.float16:
        assert (back[0, 0, 1] == 0).all()


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_a_second_prompt_over_rows_read_back(name):
    """A prompt in two parts written into the cache and read back for block-sparse
    attention over both, then tokens that attend the cache: each against 64 bits over what the cache holds."""
    B, H, N, D, bs = 2, 4, 512, 64, 64
    dt = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = (torch.randn(B, H, N, D, generator=g, device=DEV).to(dt) for _ in range(3))
    c = cache4.KVCache4(B, H, N + 8, D, dtype=dt)
    c.append(k[:, :, :200], v[:, :, :200])
    c.append(k[:, :, 200:], v[:, :, 200:])
    kr, vr = c.read(N)
    want = ref.held(k, v)
    assert torch.equal(kr.cpu().double(), want[0]) and torch.equal(vr.cpu().double(), want[1])
    sel, _ = osel.select_mean_pooled(np64(q), np64(kr), bs, 3, True, name)
    o = ops.attention_forward(q, kr, vr, torch.as_tensor(sel[:, None]).to(DEV), mask=_lib.MASK_SLOT_CAUSAL, need_lse=True)[0]
    assert_close(np64(o), oattn.fwd(np64(q), want[0].numpy(), want[1].numpy(), sel[:, None], "slot_causal")[0], name, "o")
    k1, v1, q1 = (torch.randn(B, h, 3, D, generator=g, device=DEV).to(dt) for h in (H, H, 2 * H))
    c.append(k1, v1)
    got = c.attend(q1, need_lse=True)
    ref.check_attend(got, (c.k4, c.v4, c.step), q1, [N + 3] * B)
    assert all(torch.equal(a, b) for a, b in zip(ref.values((c.k4[:, :, N:N + 3], c.v4[:, :, N:N + 3], c.step[:, :, N:N + 3])), ref.held(k1, v1)))


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("G,T", [(1, 17), (4, 6), (8, 4)])
def test_two_tiles_a_wave_keep_fp16_probabilities_in_two_numbers(D, G, T):
    """17 to 32 rows of a KV head in fp16: no probability is rounded to fp16 (the element-wise bound of 2^-16 of sum p |v|
    for the pairs; over few keys one rounding to 2^-11 passes it many times over)."""
    B, Hkv, S, dt = 4, 2, 150, torch.float16
    g = torch.Generator(device=DEV).manual_seed(D + T)
    k4, v4 = (torch.randint(0, 256, (B, Hkv, S, D // 2), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2))
    step = (0.2 + 0.3 * torch.rand(B, Hkv, S, 2, -(-D // 64), generator=g, device=DEV)).mul(64).round().div(64).to(dt)
    q = torch.randn(B, G * Hkv, T, D, generator=g, device=DEV).to(dt)
    lens = [150, 99, 40, 3]
    got = cache4.cache_attention(q, k4, v4, step, torch.tensor(lens, dtype=torch.int32, device=DEV), need_lse=True)
    r = tight.attend(q, *ref.values((k4, v4, step)), lens)
    r["big"] *= (D + 17) / (D + 4)   # (as check_attend's)
    r["a"] = r["a"] + 2.0 ** -101 * r["v1"]
    r["v1"] = torch.zeros_like(r["v1"])   # (the pairs are bf16 numbers: none of fp16's smallest parts)
    tight.check((*got, None), r, q, S, rounded=False)
