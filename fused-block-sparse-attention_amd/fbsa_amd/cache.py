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
are refused while gradients are being recorded, those with a forward-mode
tangent always. The reference attends over whole prompts only and has no
counterpart.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from .ops import _dtype_code, _ptr

# ---- layout plans -----------------------------------------------------------
# What a call checks and describes follows from its tensors' shapes, strides,
# types and device, so it is worked out once per layout: a decode loop, whose
# layouts repeat, pays for a lookup. A plan holds the C descriptor and sizes, no
# address and no value of a tensor; alignment and overlap are looked at each call.

_plans = {}
_PLANS_MAX = 1024


def _key(what, scalars, ts):
    """What a plan depends on; refuses tensors that a recorded graph, or a tangent, would need gradients of."""
    key, grad, dual = [what, scalars], torch.is_grad_enabled(), forward_ad._current_level >= 0
    for t in ts:
        if t is None:
            key.append(None)
        else:
            if (grad and t.requires_grad) or (dual and forward_ad.unpack_dual(t).tangent is not None):
                raise ValueError(f"fbsa.{what}: no gradients are formed (call it under torch.no_grad(), without forward-mode tangents)")
            key += (t.shape, t.stride(), t.dtype, t.get_device())
    return tuple(key)


def _plan(what, make, scalars, ts):
    """The plan of tensors ts (None entries allowed) for the call ``what``."""
    key = _key(what, scalars, ts)
    p = _plans.get(key)
    if p is None:
        dev = next(t.get_device() for t in ts if t is not None)
        if any(t is not None and not t.is_cuda for t in ts):
            raise ValueError(f"fbsa.{what}: tensors must be on the GPU (no CPU path)")
        if any(t is not None and t.get_device() != dev for t in ts):
            raise ValueError(f"fbsa.{what}: tensors are on different GPUs")
        p = make(what, scalars, *ts)
        p.device = torch.device("cuda", dev)
        p.index = dev
        if len(_plans) >= _PLANS_MAX:
            _plans.clear()
        _plans[key] = p
    return p


class _Plan:
    """One layout's descriptor and what the call needs besides."""


def _launch(p, fn, what, *args):
    """fn(descriptor, args..., stream) on the plan's device and its current stream."""
    if torch.cuda.current_device() != p.index:
        with torch.cuda.device(p.index):
            st = fn(p.d, *args, torch._C._cuda_getCurrentRawStream(p.index))
    else:
        st = fn(p.d, *args, torch._C._cuda_getCurrentRawStream(p.index))
    if st:
        _lib.check(st, what)


def _strides(t, n):
    """The first n strides; a dimension of one entry is never stepped along."""
    return tuple(s if e > 1 else 0 for s, e in zip(t.stride()[:n], t.shape[:n]))


def _strided(t, n):
    return t.stride(-1) == 1 and all(s * t.element_size() % 16 == 0 for s in _strides(t, n))


def _rows(what, name, t, shape, dtype, n=3):
    """A tensor of rows that the kernels address in place (caches are never copied)."""
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype:
        raise ValueError(f"fbsa.{what}: {name} must be {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")
    if t.numel() and not _strided(t, n):
        raise ValueError(f"fbsa.{what}: {name} must have contiguous rows and strides of whole 16 bytes, got {t.stride()}")


def _weights(what, name, t, shape):
    if tuple(t.shape) != tuple(shape) or t.dtype != torch.float32:
        raise ValueError(f"fbsa.{what}: {name} must be {tuple(shape)} float32, got {tuple(t.shape)} {t.dtype}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"fbsa.{what}: {name} must be contiguous along its rows, got strides {t.stride()}")


def _ints(what, name, t, B):
    if t is not None and (t.shape != (B,) or t.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"fbsa.{what}: {name} must be ({B},) int32 or int64, got {tuple(t.shape)} {t.dtype}")


def _int32(t):
    """The kernels' integers: 32 bits, contiguous; a 64-bit one beyond them is as far out as 32 bits say."""
    if t is None or (t.dtype == torch.int32 and t.is_contiguous()):
        return t
    if t.dtype != torch.int32:
        t = t.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)
    return t.contiguous()


def _bytes(t):
    """Bytes from a tensor's first entry to its last."""
    return (sum((e - 1) * s for e, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else 0


def _written(what, name, t):
    """A tensor that a kernel writes has no two of its entries in one place."""
    end = 1
    for s, e in sorted((s, e) for s, e in zip(t.stride(), t.shape) if e > 1):
        if s < end:
            raise ValueError(f"fbsa.{what}: {name} is written but its entries overlap (strides {t.stride()})")
        end = s * (e - 1) + end


def _apart(what, written, read):
    """Tensors that a kernel writes share no memory with the ones that the same
    call reads, both given as (address, bytes). (Interleaved key and value caches
    span the same addresses: of two written tensors only the start is compared.)"""
    for i, (lo, n) in enumerate(written):
        for a, m in read:
            if a < lo + n and lo < a + m:
                raise ValueError(f"fbsa.{what}: a tensor that is written overlaps one that the call reads")
        for a, m in written[:i]:
            if a == lo and n and m:
                raise ValueError(f"fbsa.{what}: two written tensors are the same buffer")


def _aligned(what, addresses):
    if addresses & 15:
        raise ValueError(f"fbsa.{what}: caches and prefixes must be 16-byte aligned")


# ---- the operators ----------------------------------------------------------


def _plan_append(what, _, k, v, k_new, v_new, start, count, weight):
    if k.dim() != 4 or k_new.dim() != 4:
        raise ValueError("fbsa.append: caches and new rows must be 4-D (B, Hkv, rows, D)")
    B, H, S, D = k.shape
    T = k_new.shape[2]
    p, d = _Plan(), _lib.AppendDesc()
    d.dtype = _dtype_code(k)
    _rows(what, "k", k, k.shape, k.dtype)
    _rows(what, "v", v, k.shape, k.dtype)
    for name, t in (("k_new", k_new), ("v_new", v_new)):
        if tuple(t.shape) != (B, H, T, D) or t.dtype != k.dtype:
            raise ValueError(f"fbsa.append: {name} must be {(B, H, T, D)} {k.dtype}, got {tuple(t.shape)} {t.dtype}")
    _written(what, "k", k)
    _written(what, "v", v)
    if weight is not None:
        _weights(what, "weight", weight, (B, H, S))
        _written(what, "weight", weight)
        d.sw[:] = _strides(weight, 2)
    _ints(what, "start", start, B)
    _ints(what, "count", count, B)
    p.ok = (_strided(k_new, 3), _strided(v_new, 3))
    p.bytes = tuple(_bytes(t) for t in (k, v, k_new, v_new))
    p.empty = T == 0 or B == 0
    d.B, d.H, d.T, d.S, d.D = B, H, T, S, D
    d.sk[:], d.sv[:] = _strides(k, 3), _strides(v, 3)
    packed = (H * T * D, T * D, D)
    d.skn[:] = _strides(k_new, 3) if p.ok[0] else packed
    d.svn[:] = _strides(v_new, 3) if p.ok[1] else packed
    p.d, p.packed = d, packed
    return p


def append(k, v, k_new, v_new, start, *, count=None, weight=None):
    """Writes k_new, v_new (B, Hkv, T, D) into the caches k, v (B, Hkv, S, D) at
    rows start[b] + t, for t < count[b] where a padded batch gives counts, and
    zeroes ``weight`` (B, Hkv, S) fp32 there. Rows that would fall outside the
    cache are dropped; no other row changes. ``start`` is not advanced."""
    p = _plan("append", _plan_append, (), (k, v, k_new, v_new, start, count, weight))
    if p.empty:
        return
    if (k_new.data_ptr() | v_new.data_ptr()) & 15 or not (p.ok[0] and p.ok[1]):
        k_new, v_new = (t.clone(memory_format=torch.contiguous_format) for t in (k_new, v_new))
        return append(k, v, k_new, v_new, start, count=count, weight=weight)
    nk, nv, nkn, nvn = p.bytes
    pk, pv, pkn, pvn = k.data_ptr(), v.data_ptr(), k_new.data_ptr(), v_new.data_ptr()
    _aligned("append", pk | pv)
    _apart("append", ((pk, nk), (pv, nv)), ((pkn, nkn), (pvn, nvn)))
    start, count = _int32(start), _int32(count)
    _launch(p, _lib.load().fbsa_cache_append, "fbsa_cache_append", pk, pv, pkn, pvn, start.data_ptr(), _ptr(count), _ptr(weight))
    # (what a kernel writes through an address counts as modified in place, as torch's own operations do)
    increment_version((k, v) if weight is None else (k, v, weight))


def _plan_attend(what, scalars, q, kp, vp, k, v, lens, count, out_gate, weight, out_weight):
    scale, = scalars
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"fbsa.{what}: q and the caches must be 4-D")
    B, Hq, T, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    dt = q.dtype
    p, d = _Plan(), _lib.CacheDesc()
    d.dtype = _dtype_code(q)
    _rows(what, "k", k, (B, Hkv, S, D), dt)
    _rows(what, "v", v, (B, Hkv, S, D), dt)
    p.P = 0
    if kp is not None:
        if kp.dim() != 3:
            raise ValueError(f"fbsa.{what}: the prefix must be 3-D (Hkv, P, D)")
        p.P = kp.shape[1]
        _rows(what, "k_prefix", kp, (Hkv, p.P, D), dt, 2)
        _rows(what, "v_prefix", vp, (Hkv, p.P, D), dt, 2)
        if p.P:
            d.skp[:], d.svp[:] = _strides(kp, 2), _strides(vp, 2)
    if out_gate is not None:
        if out_gate.shape != q.shape or out_gate.dtype != dt:
            raise ValueError(f"fbsa.{what}: out_gate must match q's shape and dtype")
        p.gate_ok = out_gate.stride(-1) == 1
        d.sog[:] = _strides(out_gate, 3) if p.gate_ok else (Hq * T * D, T * D, D)
    if out_weight is not None:
        _weights(what, "out_weight", out_weight, (B, Hkv, S))
        _written(what, "out_weight", out_weight)
        d.flags = _lib.CACHE_WEIGHT
        d.swo[:] = _strides(out_weight, 2)
        p.same = weight is not None and weight.stride() == out_weight.stride()
        p.bytes = (_bytes(out_weight), _bytes(weight) if weight is not None else 0)
    if weight is not None:
        _weights(what, "weight", weight, (B, Hkv, S))
        d.sw[:] = _strides(weight, 2)
    _ints(what, "lens", lens, B)
    _ints(what, "count", count, B)
    p.q_ok = _strided(q, 3)
    p.empty = q.numel() == 0
    p.shape, p.S = (B, Hq, T, D), S
    packed = (Hq * T * D, T * D, D)
    d.B, d.Hq, d.Hkv, d.T, d.S, d.P, d.D = B, Hq, Hkv, T, S, p.P, D
    d.scale = D ** -0.5 if scale is None else scale
    d.sq[:] = _strides(q, 3) if p.q_ok else packed
    d.sk[:], d.sv[:], d.so[:] = _strides(k, 3), _strides(v, 3), packed
    p.d = d
    p.nbytes = 0 if p.empty else _lib.load().fbsa_cache_attn_workspace_bytes(d)
    if p.nbytes == 0 and not p.empty:
        _lib.check(_lib.EINVAL, f"fbsa_cache_attn ({what})")
    return p


def _attend(what, q, kp, vp, k, v, lens, count, scale, out_gate, weight, out_weight, need_lse):
    if out_weight is None:
        out_weight = weight
    scale = None if scale is None else float(scale)
    p = _plan(what, _plan_attend, (scale,), (q, kp, vp, k, v, lens, count, out_gate, weight, out_weight))
    o = torch.empty(p.shape, dtype=q.dtype, device=p.device)
    lse = torch.empty(p.shape[:3], dtype=torch.float32, device=p.device) if need_lse else None
    if p.empty:
        if out_weight is not None and out_weight is not weight and out_weight.numel():
            raise ValueError(f"fbsa.{what}: no queries to take weights from")
        return (o, lse) if need_lse else o
    if q.data_ptr() & 15 or not p.q_ok:
        q = q.clone(memory_format=torch.contiguous_format)
        if p.q_ok:  # (the plan describes the tensor that was given)
            return _attend(what, q, kp, vp, k, v, lens, count, scale, out_gate, weight, out_weight, need_lse)
    if out_gate is not None and not p.gate_ok:
        out_gate = out_gate.clone(memory_format=torch.contiguous_format)
    pk, pv = k.data_ptr(), v.data_ptr()
    pkp, pvp = (kp.data_ptr(), vp.data_ptr()) if p.P else (None, None)
    _aligned(what, pk | pv | pkp | pvp if p.P else pk | pv)
    pw, pwo = _ptr(weight), _ptr(out_weight)
    if pw is not None and not (p.same and pw == pwo):
        _apart(what, ((pwo, p.bytes[0]),), ((pw, p.bytes[1]),))
    lens = torch.full(p.shape[:1], p.S, dtype=torch.int32, device=p.device) if lens is None else _int32(lens)
    count = _int32(count)
    ws = torch.empty(p.nbytes, dtype=torch.uint8, device=p.device)
    _launch(p, _lib.load().fbsa_cache_attn, what, q.data_ptr(), pk, pv, lens.data_ptr(), _ptr(count), pkp, pvp,
            _ptr(out_gate), o.data_ptr(), _ptr(lse), pw, pwo, ws.data_ptr(), p.nbytes)
    if out_weight is not None:
        increment_version(out_weight)
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
    from zeros. No new tokens (T = 0) leave weight itself as it is; another
    out_weight is refused then.

    Returns o (B, Hq, T, D), and with need_lse the fp32 natural-log normaliser
    (B, Hq, T); padding queries, and queries that see no row or whose every score
    is -inf, give 0 and -inf, and no weight.
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


def _plan_evict(what, scalars, k, v, weight, lens, ko, vo, wo):
    budget, recent, sink = scalars
    if k.dim() != 4:
        raise ValueError("fbsa.evict: caches must be 4-D (B, Hkv, S, D)")
    B, H, S, D = k.shape
    p, d = _Plan(), _lib.EvictDesc()
    d.dtype = _dtype_code(k)
    _rows(what, "k", k, k.shape, k.dtype)
    _rows(what, "v", v, k.shape, k.dtype)
    _weights(what, "weight", weight, (B, H, S))
    _ints(what, "lens", lens, B)
    inplace = ko is None
    if inplace:
        d.flags = _lib.EVICT_IN_PLACE
        ko, vo, wo = k, v, weight
    SO = ko.shape[2] if ko.dim() == 4 else 0
    _rows(what, "k_out", ko, (B, H, SO, D), k.dtype)
    _rows(what, "v_out", vo, (B, H, SO, D), k.dtype)
    _weights(what, "weight_out", wo, (B, H, SO))
    for name, t in (("k", ko), ("v", vo), ("weight", wo)):
        _written(what, name, t)
    d.B, d.H, d.S, d.SO, d.D, d.budget, d.recent, d.sink = B, H, S, SO, D, budget, recent, sink
    d.sk[:], d.sv[:], d.sko[:], d.svo[:] = _strides(k, 3), _strides(v, 3), _strides(ko, 3), _strides(vo, 3)
    d.sw[:], d.swo[:] = _strides(weight, 2), _strides(wo, 2)
    p.d, p.inplace = d, inplace
    p.B, p.shape = B, (B, H, max(0, min(budget, S)))
    p.bytes = tuple(_bytes(t) for t in (k, v, weight, ko, vo, wo))
    p.nbytes = _lib.load().fbsa_cache_evict_workspace_bytes(d)
    return p


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
    ko, vo, wo = out if out is not None else (None, None, None)
    if out is not None and any(t is None for t in out):
        raise ValueError("fbsa.evict: out must be (k_out, v_out, weight_out)")
    p = _plan("evict", _plan_evict, (int(budget), int(recent), int(sink)), (k, v, weight, lens, ko, vo, wo))
    pk, pv, pw = k.data_ptr(), v.data_ptr(), weight.data_ptr()
    if p.inplace:
        pko, pvo, pwo = pk, pv, pw
    else:
        pko, pvo, pwo = ko.data_ptr(), vo.data_ptr(), wo.data_ptr()
        nk, nv, nw, nko, nvo, nwo = p.bytes
        _apart("evict", ((pko, nko), (pvo, nvo), (pwo, nwo)), ((pk, nk), (pv, nv), (pw, nw)))
    if pk == pv:
        raise ValueError("fbsa.evict: the key and value caches are the same buffer")
    _aligned("evict", pk | pv | pko | pvo)
    lens = _int32(lens)
    index = torch.empty(p.shape, dtype=torch.int32, device=p.device)
    new_lens = torch.empty(p.B, dtype=torch.int32, device=p.device)
    ws = torch.empty(p.nbytes, dtype=torch.uint8, device=p.device) if p.nbytes else None
    _launch(p, _lib.load().fbsa_cache_evict, "fbsa_cache_evict", pk, pv, pw, lens.data_ptr(), pko, pvo, pwo, index.data_ptr(),
            new_lens.data_ptr(), _ptr(ws), p.nbytes)
    increment_version((k, v, weight) if p.inplace else (ko, vo, wo))
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
