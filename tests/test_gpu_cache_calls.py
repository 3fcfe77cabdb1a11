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


def test_what_a_call_writes_counts_as_modified():
    q, k, v, _, _, g = _make("bf16", 1, 4, 2, 1, 40, 64, [40])
    w, lens = _randn(g, 1, 2, 40).abs(), _ints([40])
    losses = [_saved(x) for x in (k, v, w)]
    cache.append(k, v, q[:, :2], q[:, :2], _ints([3]), weight=w)
    for x in losses:
        _raises(x)
    a, b, out = _saved(k), _saved(w), torch.zeros_like(w)
    c = _saved(out)
    cache.cache_attention(q, k, v, lens, weight=w, out_weight=out)
    a.backward()
    b.backward()
    _raises(c)
    c = _saved(w)
    cache.cache_attention(q, k, v, lens, weight=w)
    _raises(c)
    dst = [torch.zeros(1, 2, 8, 64, dtype=k.dtype, device=DEV) for _ in range(2)] + [torch.zeros(1, 2, 8, device=DEV)]
    losses, kept = [_saved(x) for x in dst], [_saved(x) for x in (k, v, w)]
    cache.evict(k, v, w, lens, 8, out=dst)
    for x in losses:
        _raises(x)
    for x in kept:
        x.backward()
    losses = [_saved(x) for x in (k, v, w)]
    cache.evict(k, v, w, lens, 8)
    for x in losses:
        _raises(x)


def test_caches_made_in_inference_mode():
    with torch.inference_mode():
        c = cache.KVCache(2, 2, 64, 64, weight=True)
        x = _randn(_gen(0), 2, 2, 3, 64, dtype=torch.bfloat16)
        c.append(x, x)
        c.attend(x)
        c.evict(2)
    assert c.lens.tolist() == [2, 2]


def test_no_new_tokens():
    g = _gen(0)
    for weight in (False, True):
        c = cache.KVCache(2, 2, 64, 64, weight=weight)
        c.append(*(_randn(g, 2, 2, 5, 64, dtype=torch.bfloat16) for _ in range(2)))
        none = torch.zeros(2, 4, 0, 64, dtype=torch.bfloat16, device=DEV)
        if weight:
            c.weight.copy_(_randn(g, 2, 2, 64))
            before = c.weight.clone()
        c.append(none[:, :2], none[:, :2])
        o, lse = c.attend(none, need_lse=True)
        assert o.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0) and c.lens.tolist() == [5, 5]
        if weight:
            assert torch.equal(c.weight, before)
            with pytest.raises(ValueError, match="no queries"):   # nothing would fill another tensor
                cache.cache_attention(none, c.k, c.v, c.lens, weight=c.weight, out_weight=torch.zeros_like(c.weight))
