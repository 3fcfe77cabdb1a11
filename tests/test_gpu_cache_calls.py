"""Calls of the cache operators that meet the rest of a program: 64-bit lengths,
tensors that autograd has saved, no new tokens."""
import pytest
import torch

from fbsa_amd import cache
from test_gpu_cache import DEV, _gen, _ints, _make, _randn

pytestmark = pytest.mark.gpu


def test_lengths_and_places_beyond_32_bits():
    q, k, v, _, _, g = _make("bf16", 2, 4, 2, 1, 40, 64, [40, 40])
    far = torch.tensor([1 << 32, (1 << 33) + 3], device=DEV)
    before = k.clone(), v.clone()
    cache.append(k, v, q[:, :2], q[:, :2], far)
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    cache.append(k, v, q[:, :2], q[:, :2], _ints([0, 0]), count=-far)
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    assert torch.equal(cache.cache_attention(q, k, v, far), cache.cache_attention(q, k, v))
    assert (cache.cache_attention(q, k, v, -far) == 0).all()
    w, out = _randn(g, 2, 2, 40), [torch.zeros(2, 2, 8, 64, dtype=k.dtype, device=DEV) for _ in range(2)]
    index, n = cache.evict(k, v, w, far, 8, out=(*out, torch.zeros(2, 2, 8, device=DEV)))
    assert n.tolist() == [8, 8] and torch.equal(index, cache.evict(k, v, w, _ints([40, 40]), 8)[0])


def _saved(t):
    """A loss whose backward needs t as it is now."""
    return (torch.ones_like(t, requires_grad=True) * t).sum()


def _raises(loss):
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
