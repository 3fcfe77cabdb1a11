"""Caches of keys and values over the C ABI (gfx950): what serving does after a prompt.

A cache holds B sequences: k, v (B, Hkv, S, D) of capacity S, sequence b's rows
being [0, lens[b]), in any layout whose rows are contiguous and whose strides
are multiples of 16 bytes; D is a multiple of 8 up to 256. ``lens``, ``start``
and ``count`` are (B,) integer tensors on the GPU that the kernels read, so no
call synchronises and a captured graph follows their values.

* ``append``                   writes new rows behind each sequence
* ``cache_attention``          the newest tokens over their sequence's rows
* ``shared_prefix_attention``  the same behind a prefix held once for the batch
* ``evict``                    cuts each sequence to a budget of rows by the
                               attention weight that they gathered
* ``KVCache``                  the four over one set of buffers

They are for inference: no gradients are formed, and inputs that require grad
are refused while gradients are being recorded. The reference attends over
whole prompts only and has no counterpart.
"""
import torch

from . import _lib
from .ops import _dtype_code, _kernel_ready, _ptr, _require_cuda, _stream


def _check(what, *ts):
    """On one GPU, and not part of a graph that would need their gradients."""
    ts = [t for t in ts if t is not None]
    _require_cuda(*ts)
    if any(t.device != ts[0].device for t in ts):
        raise ValueError(f"fbsa.{what}: tensors are on different GPUs")
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise ValueError(f"fbsa.{what}: no gradients are formed (call it under torch.no_grad())")


def _strides(t, n):
    """The first n strides; a dimension of one entry is never stepped along."""
    return tuple(s if e > 1 else 0 for s, e in zip(t.stride()[:n], t.shape[:n]))


def _rows(what, name, t, shape, dtype, n=3):
    """A tensor of rows that the kernels address in place (caches are never copied)."""
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype:
        raise ValueError(f"fbsa.{what}: {name} must be {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")
    es = t.element_size()
    if t.numel() and (t.stride(-1) != 1 or t.data_ptr() % 16 or any((s * es) % 16 for s in _strides(t, n))):
        raise ValueError(f"fbsa.{what}: {name} must have contiguous rows and 16-byte aligned strides, got {t.stride()}")
    return t


def _weights(what, name, t, shape):
    if tuple(t.shape) != tuple(shape) or t.dtype != torch.float32:
        raise ValueError(f"fbsa.{what}: {name} must be {tuple(shape)} float32, got {tuple(t.shape)} {t.dtype}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"fbsa.{what}: {name} must be contiguous along its rows, got strides {t.stride()}")
    return t


def _ints(what, name, t, B):
    if t.shape != (B,) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"fbsa.{what}: {name} must be ({B},) int32 or int64, got {tuple(t.shape)} {t.dtype}")
    return t.to(torch.int32).contiguous()


def _span(t):
    return t.data_ptr(), t.data_ptr() + (sum((e - 1) * s for e, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _written(what, name, t, *others):
    """A tensor that a kernel writes: no two of its entries in one place, and
    apart from the tensors that the same call reads."""
    end = 1
    for s, e in sorted((s, e) for s, e in zip(t.stride(), t.shape) if e > 1):
        if s < end:
            raise ValueError(f"fbsa.{what}: {name} is written but its entries overlap (strides {t.stride()})")
        end = s * (e - 1) + end
    lo, hi = _span(t)
    for x in others:
        if x is not None and t.numel() and x.numel():
            a, b = _span(x)
            if a < hi and lo < b:
                raise ValueError(f"fbsa.{what}: {name} is written but overlaps a tensor that the call reads")


def _apart(what, k, v):
    # (interleaved caches span the same addresses, so only the plain mistake is seen here)
    if k.numel() and k.data_ptr() == v.data_ptr():
        raise ValueError(f"fbsa.{what}: the key and value caches are the same buffer")


def append(k, v, k_new, v_new, start, *, count=None, weight=None):
    """Writes k_new, v_new (B, Hkv, T, D) into the caches k, v (B, Hkv, S, D) at
    rows start[b] + t, for t < count[b] where a padded batch gives counts, and
    zeroes ``weight`` (B, Hkv, S) fp32 there. Rows that would fall outside the
    cache are dropped; no other row changes. ``start`` is not advanced."""
    _check("append", k, v, k_new, v_new, start, count, weight)
    if k.dim() != 4 or k_new.dim() != 4:
        raise ValueError("fbsa.append: caches and new rows must be 4-D (B, Hkv, rows, D)")
    B, H, S, D = k.shape
    T = k_new.shape[2]
    d = _lib.AppendDesc()
    d.dtype = _dtype_code(k)
    _rows("append", "k", k, k.shape, k.dtype)
    _rows("append", "v", v, k.shape, k.dtype)
    for name, t in (("k_new", k_new), ("v_new", v_new)):
        if tuple(t.shape) != (B, H, T, D) or t.dtype != k.dtype:
            raise ValueError(f"fbsa.append: {name} must be {(B, H, T, D)} {k.dtype}, got {tuple(t.shape)} {t.dtype}")
    _written("append", "k", k, k_new, v_new)
    _written("append", "v", v, k_new, v_new)
    _apart("append", k, v)
    if weight is not None:
        _weights("append", "weight", weight, (B, H, S))
        _written("append", "weight", weight)
    start = _ints("append", "start", start, B)
    count = None if count is None else _ints("append", "count", count, B)
    if T == 0 or B == 0:
        return
    new = [_kernel_ready(t) for t in (k_new, v_new)]
    d.B, d.H, d.T, d.S, d.D = B, H, T, S, D
    d.sk[:], d.sv[:], d.skn[:], d.svn[:] = _strides(k, 3), _strides(v, 3), _strides(new[0], 3), _strides(new[1], 3)
    d.sw[:] = (0, 0) if weight is None else _strides(weight, 2)
    with torch.cuda.device(k.device):
        _lib.check(_lib.load().fbsa_cache_append(d, _ptr(k), _ptr(v), _ptr(new[0]), _ptr(new[1]), _ptr(start), _ptr(count),
                                                 _ptr(weight), _stream()), "fbsa_cache_append")


def _attend(what, q, kp, vp, k, v, lens, count, scale, out_gate, weight, out_weight, need_lse):
    _check(what, q, kp, vp, k, v, lens, count, out_gate, weight, out_weight)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"fbsa.{what}: q and the caches must be 4-D")
    B, Hq, T, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    dt = q.dtype
    code = _dtype_code(q)
    _rows(what, "k", k, (B, Hkv, S, D), dt)
    _rows(what, "v", v, (B, Hkv, S, D), dt)
    P = 0
    if kp is not None:
        if kp.dim() != 3:
            raise ValueError(f"fbsa.{what}: the prefix must be 3-D (Hkv, P, D)")
        P = kp.shape[1]
        _rows(what, "k_prefix", kp, (Hkv, P, D), dt, 2)
        _rows(what, "v_prefix", vp, (Hkv, P, D), dt, 2)
    if out_gate is not None and (out_gate.shape != q.shape or out_gate.dtype != dt):
        raise ValueError(f"fbsa.{what}: out_gate must match q's shape and dtype")
    if out_weight is None:
        out_weight = weight
    if out_weight is not None:
        _weights(what, "out_weight", out_weight, (B, Hkv, S))
        same = weight is not None and weight.data_ptr() == out_weight.data_ptr() and weight.stride() == out_weight.stride()
        if weight is not None:
            _weights(what, "weight", weight, (B, Hkv, S))
        _written(what, "out_weight", out_weight, None if same else weight)
    lens = (torch.full((B,), S, dtype=torch.int32, device=q.device) if lens is None else _ints(what, "lens", lens, B))
    count = None if count is None else _ints(what, "count", count, B)
    if q.numel() == 0:
        if out_weight is not None and B:
            raise ValueError(f"fbsa.{what}: no queries to take weights from")
        o, lse = torch.empty_like(q), torch.empty(B, Hq, T, dtype=torch.float32, device=q.device)
        return (o, lse) if need_lse else o
    q = _kernel_ready(q)
    og = out_gate
    if og is not None and og.stride(-1) != 1:
        og = og.contiguous()
    o = torch.empty(B, Hq, T, D, dtype=dt, device=q.device)
    lse = torch.empty(B, Hq, T, dtype=torch.float32, device=q.device) if need_lse else None
    d = _lib.CacheDesc()
    d.dtype = code
    d.B, d.Hq, d.Hkv, d.T, d.S, d.P, d.D = B, Hq, Hkv, T, S, P, D
    d.scale = float(D ** -0.5 if scale is None else scale)
    d.sq[:], d.sk[:], d.sv[:], d.so[:] = _strides(q, 3), _strides(k, 3), _strides(v, 3), _strides(o, 3)
    d.sog[:] = (0, 0, 0) if og is None else _strides(og, 3)
    if P:
        d.skp[:], d.svp[:] = _strides(kp, 2), _strides(vp, 2)
    if weight is not None:
        d.sw[:] = _strides(weight, 2)
    if out_weight is not None:
        d.flags = _lib.CACHE_WEIGHT
        d.swo[:] = _strides(out_weight, 2)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        nbytes = lib.fbsa_cache_attn_workspace_bytes(d)
        if nbytes == 0:
            _lib.check(_lib.EINVAL, f"fbsa_cache_attn ({what})")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        _lib.check(lib.fbsa_cache_attn(d, _ptr(q), _ptr(k), _ptr(v), _ptr(lens), _ptr(count), _ptr(kp) if P else None,
                                       _ptr(vp) if P else None, _ptr(og), _ptr(o), _ptr(lse), _ptr(weight), _ptr(out_weight),
                                       _ptr(ws), nbytes, _stream()), f"fbsa_cache_attn ({what})")
    return (o, lse) if need_lse else o


def cache_attention(q, k, v, lens=None, *, count=None, scale=None, out_gate=None, weight=None, out_weight=None,
                    need_lse=False):
    """Attention of each sequence's newest tokens over its cache.

    q (B, Hq, T, D); k, v (B, Hkv, S, D), query head h reading KV head
    h // (Hq // Hkv); lens (B,) rows per sequence, the new tokens' own rows
    among them (default: S). Query t of a sequence is the token of row
    lens - T + t and sees the rows up to its own; in a padded batch ``count``
    (B,) says how many of the T queries are real: query t < count is the token
    of row lens - count + t, the others are padding. out_gate (B, Hq, T, D):
    o <- o * sigmoid(out_gate).

    weight (B, Hkv, S) fp32, the attention weight that each row has gathered:
    out_weight (default: weight itself) receives weight plus the probability
    that these queries, summed over the group's heads, gave each row below
    lens; rows at or past lens are left as they were. out_weight alone starts
    from zeros.

    Returns o (B, Hq, T, D), and with need_lse the fp32 natural-log normaliser
    (B, Hq, T); padding queries, and queries that see no row, give 0 and -inf.
    """
    return _attend("cache_attention", q, None, None, k, v, lens, count, scale, out_gate, weight, out_weight, need_lse)


def shared_prefix_attention(q, k_prefix, v_prefix, k, v, lens=None, *, count=None, scale=None, out_gate=None, weight=None,
                            out_weight=None, need_lse=False):
    """``cache_attention`` where every sequence continues the same P rows.

    k_prefix, v_prefix (Hkv, P, D) stand before every sequence's own rows k, v
    (B, Hkv, S, D): each real query sees all of them and its own rows as above,
    in one softmax. The prefix is read once for the whole batch, its products
    taken over the stacked queries of all sequences. Weights are kept for the
    own rows only.
    """
    if k_prefix is None or v_prefix is None:
        raise ValueError("fbsa.shared_prefix_attention: k_prefix and v_prefix are required")
    return _attend("shared_prefix_attention", q, k_prefix, v_prefix, k, v, lens, count, scale, out_gate, weight,
                   out_weight, need_lse)


def evict(k, v, weight, lens, budget, *, recent=0, sink=0, out=None):
    """Cuts every sequence of a cache to at most ``budget`` rows per head.

    A sequence longer than budget keeps its first ``sink`` rows, its last
    ``recent`` rows and, of those between, the budget - sink - recent of greatest
    accumulated ``weight`` (B, Hkv, S) fp32 (ties to the lower row, NaN ranks as
    -inf). Kept rows keep their order. k, v and weight move within their own
    buffers, or with out = (k_out, v_out, weight_out) of capacity
    >= min(budget, S) into those. Rows past a sequence's new length are left as they were
    in the outputs.

    Returns (index, new_lens): index (B, Hkv, min(budget, S)) int32, the row that
    each kept row had (-1 past the last); new_lens (B,) int32 = min(lens, budget).
    ``lens`` itself does not change.
    """
    _check("evict", k, v, weight, lens, *(out or ()))
    if k.dim() != 4:
        raise ValueError("fbsa.evict: caches must be 4-D (B, Hkv, S, D)")
    B, H, S, D = k.shape
    d = _lib.EvictDesc()
    d.dtype = _dtype_code(k)
    _rows("evict", "k", k, k.shape, k.dtype)
    _rows("evict", "v", v, k.shape, k.dtype)
    _weights("evict", "weight", weight, (B, H, S))
    lens = _ints("evict", "lens", lens, B)
    budget, recent, sink = int(budget), int(recent), int(sink)
    if out is None:
        d.flags = _lib.EVICT_IN_PLACE
        ko, vo, wo = k, v, weight
        others = ()
    else:
        ko, vo, wo = out
        others = (k, v, weight)
    SO = ko.shape[2] if ko.dim() == 4 else 0
    _rows("evict", "k_out", ko, (B, H, SO, D), k.dtype)
    _rows("evict", "v_out", vo, (B, H, SO, D), k.dtype)
    _weights("evict", "weight_out", wo, (B, H, SO))
    for name, t in (("k", ko), ("v", vo), ("weight", wo)):
        _written("evict", name, t, *others)
    _apart("evict", ko, vo)
    index = torch.empty(B, H, max(0, min(budget, S)), dtype=torch.int32, device=k.device)
    new_lens = torch.empty(B, dtype=torch.int32, device=k.device)
    d.B, d.H, d.S, d.SO, d.D, d.budget, d.recent, d.sink = B, H, S, SO, D, budget, recent, sink
    d.sk[:], d.sv[:], d.sko[:], d.svo[:] = _strides(k, 3), _strides(v, 3), _strides(ko, 3), _strides(vo, 3)
    d.sw[:], d.swo[:] = _strides(weight, 2), _strides(wo, 2)
    lib = _lib.load()
    with torch.cuda.device(k.device):
        nbytes = lib.fbsa_cache_evict_workspace_bytes(d)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=k.device) if nbytes else None
        _lib.check(lib.fbsa_cache_evict(d, _ptr(k), _ptr(v), _ptr(weight), _ptr(lens), _ptr(ko), _ptr(vo), _ptr(wo), _ptr(index),
                                        _ptr(new_lens), _ptr(ws), nbytes, _stream()), "fbsa_cache_evict")
    return index, new_lens


class KVCache:
    """One layer's cache of B sequences and the calls of a decode loop over it.

    Buffers k, v (B, Hkv, S, D), lens (B,) int32 and, with weight=True, the
    accumulated weights (B, Hkv, S) are the object's; all calls stay on the
    device. The caller keeps every sequence within S rows (``evict`` first):
    rows past the capacity are dropped by ``append``.
    """

    def __init__(self, B, Hkv, S, D, *, dtype=torch.bfloat16, device="cuda", weight=False):
        self.k = torch.zeros(B, Hkv, S, D, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.lens = torch.zeros(B, dtype=torch.int32, device=device)
        self.weight = torch.zeros(B, Hkv, S, dtype=torch.float32, device=device) if weight else None

    def append(self, k_new, v_new, count=None):
        """New rows (B, Hkv, T, D) behind every sequence (count[b] of them in a padded batch)."""
        append(self.k, self.v, k_new, v_new, self.lens, count=count, weight=self.weight)
        grow = k_new.shape[2] if count is None else count.clamp(0, k_new.shape[2])
        self.lens.add_(grow).clamp_(max=self.k.shape[2])

    def attend(self, q, *, prefix=None, count=None, scale=None, out_gate=None, need_lse=False):
        """Attention of the rows just appended; prefix: (k_prefix, v_prefix) that
        every sequence continues. Adds to the weights where they are kept."""
        kp, vp = (None, None) if prefix is None else prefix
        what = "cache_attention" if prefix is None else "shared_prefix_attention"
        return _attend(what, q, kp, vp, self.k, self.v, self.lens, count, scale, out_gate, self.weight, None, need_lse)

    def evict(self, budget, *, recent=0, sink=0):
        """Cuts every sequence to ``budget`` rows in place; returns the rows kept (``evict``)."""
        if self.weight is None:
            raise ValueError("fbsa.KVCache: eviction needs the weights (weight=True)")
        index, lens = evict(self.k, self.v, self.weight, self.lens, budget, recent=recent, sink=sink)
        self.lens.copy_(lens)
        return index
