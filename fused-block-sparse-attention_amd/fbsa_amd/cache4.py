"""Caches of keys and values held in 4 bits, over the C ABI (gfx950).

A cache is three tensors: ``k4``, ``v4`` (B, Hkv, S, D / 2) uint8, two codes to a
byte (element 2i in the low half), and ``step`` (B, Hkv, S, 2, ng), ng =
ceil(D / 64): the steps of a row's key, then of its value, one for each 64
elements (the last 32 where D is an odd multiple of 32). A value is step * code,
code a 4-bit float (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign); step is the group's
largest magnitude over 6, rounded to 6 significant bits, so every value is a
number of the rows' type exactly. Steps are fp16 for fp16 rows and bf16 for bf16
and fp32 ones. 4.25 bits a value where D is a multiple of 64. D is a multiple of
32 up to 256; the codes may lie in any layout whose rows are contiguous and whose
strides are multiples of 16 bytes, each (sequence, head)'s steps are contiguous.

* ``append``           quantises new rows behind each sequence
* ``read``             rows back as numbers, exactly what attention sees
* ``cache_attention``  the newest tokens over their sequence's rows
* ``empty``            the three tensors
* ``KVCache4``         the calls over one set of them

``lens``, ``start``, ``first`` and ``count`` are (B,) integer tensors on the GPU,
as in ``cache``; nothing synchronises. For inference: inputs that require grad are
refused while gradients are being recorded, those with a forward-mode tangent
always. The reference keeps no caches and has no counterpart.
"""
import torch
from torch.autograd.graph import increment_version

from . import _lib
from .cache import _Plan, _aligned, _apart, _bytes, _int32, _ints, _launch, _plan, _rows, _strided, _strides, _written
from .ops import _dtype_code, _ptr

GROUP = 64  # elements to a step


def _step_type(dtype):
    return torch.float16 if dtype == torch.float16 else torch.bfloat16


def empty(B, Hkv, S, D, *, dtype=torch.bfloat16, device="cuda"):
    """(k4, v4, step) of a cache for rows of type ``dtype``; every row reads as zeros."""
    if D % 32 or not 32 <= D <= 256:
        raise ValueError(f"fbsa.cache4: head dim {D} is not a multiple of 32 up to 256")
    k4 = torch.zeros(B, Hkv, S, D // 2, dtype=torch.uint8, device=device)
    step = torch.zeros(B, Hkv, S, 2, -(-D // GROUP), dtype=_step_type(dtype), device=device)
    return k4, torch.zeros_like(k4), step


def _held(what, d, k4, v4, step, dtype):
    """Checks a cache's tensors and describes them; (B, Hkv, S, D)."""
    if k4.dim() != 4:
        raise ValueError(f"fbsa.{what}: codes must be 4-D (B, Hkv, rows, D / 2)")
    B, H, S, half = k4.shape
    D = 2 * half
    _rows(what, "k4", k4, k4.shape, torch.uint8)
    _rows(what, "v4", v4, k4.shape, torch.uint8)
    ng = -(-D // GROUP)
    if tuple(step.shape) != (B, H, S, 2, ng) or step.dtype != _step_type(dtype):
        raise ValueError(f"fbsa.{what}: step must be {(B, H, S, 2, ng)} {_step_type(dtype)}, got {tuple(step.shape)} {step.dtype}")
    for s, want, e in zip(step.stride()[2:], (2 * ng, ng, 1), step.shape[2:]):
        if e > 1 and s != want:
            raise ValueError(f"fbsa.{what}: each head's steps must be contiguous, got strides {step.stride()}")
    ss = _strides(step, 2)
    if any(s % 2 for s in ss):
        raise ValueError(f"fbsa.{what}: strides of the steps must be even, got {step.stride()}")
    d.sk4[:], d.sv4[:], d.ss[:] = _strides(k4, 3), _strides(v4, 3), ss
    return B, H, S, D


def _plan_rows(what, scalars, k4, v4, step, k, v, first, count):
    T, dtype = scalars
    p, d = _Plan(), _lib.Rows4Desc()
    B, H, S, D = _held(what, d, k4, v4, step, dtype)
    for name, t in (("k", k), ("v", v)):
        if t is not None and (tuple(t.shape) != (B, H, T, D) or t.dtype != dtype):
            raise ValueError(f"fbsa.{what}: {name} must be {(B, H, T, D)} {dtype}, got {tuple(t.shape)} {t.dtype}")
    _ints(what, "first" if what == "cache4.read" else "start", first, B)
    _ints(what, "count", count, B)
    d.dtype = _dtype_code(torch.empty(0, dtype=dtype))
    d.B, d.H, d.T, d.S, d.D = B, H, T, S, D
    packed = (H * T * D, T * D, D)
    p.ok = tuple(t is None or _strided(t, 3) for t in (k, v))
    d.sk[:] = _strides(k, 3) if k is not None and p.ok[0] else packed
    d.sv[:] = _strides(v, 3) if v is not None and p.ok[1] else packed
    if what == "cache4.append":
        for name, t in (("k4", k4), ("v4", v4), ("step", step)):
            _written(what, name, t)
    elif k is not None:
        for name, t, ok in zip("kv", (k, v), p.ok):
            if t.numel() and not ok:
                raise ValueError(f"fbsa.{what}: {name} must have contiguous rows and strides of whole 16 bytes, got {t.stride()}")
            _written(what, name, t)
    p.empty = B == 0 or H == 0 or T == 0 or S == 0
    p.shape = (B, H, T, D)
    p.bytes = tuple(0 if t is None else _bytes(t) for t in (k4, v4, step, k, v))
    p.d = d
    return p


def append(k4, v4, step, k_new, v_new, start, *, count=None):
    """Quantises k_new, v_new (B, Hkv, T, D) into the cache at rows start[b] + t, for
    t < count[b] where a padded batch gives counts. Rows that would fall outside the
    cache are dropped; no other row changes. ``start`` is not advanced. A row whose key
    or value holds a NaN or an infinity (one head's) is held as NaN, key and value."""
    if k_new.dim() != 4:
        raise ValueError("fbsa.cache4.append: new rows must be 4-D (B, Hkv, rows, D)")
    if start is None:
        raise ValueError("fbsa.cache4.append: start is required")
    p = _plan("cache4.append", _plan_rows, (k_new.shape[2], k_new.dtype), (k4, v4, step, k_new, v_new, start, count))
    if p.empty:
        return
    at = (k4.data_ptr(), v4.data_ptr(), step.data_ptr(), k_new.data_ptr(), v_new.data_ptr())
    if (at[3] | at[4]) & 15 or not (p.ok[0] and p.ok[1]):
        k_new, v_new = (t.clone(memory_format=torch.contiguous_format) for t in (k_new, v_new))
        return append(k4, v4, step, k_new, v_new, start, count=count)
    _aligned("cache4.append", at[0] | at[1])
    spans = tuple(zip(at, p.bytes))
    _apart("cache4.append", spans[:3], spans[3:])
    start, count = _int32(start), _int32(count)
    _launch(p, _lib.load().fbsa_cache4_append, "fbsa_cache4_append", *at, start.data_ptr(), _ptr(count))
    increment_version((k4, v4, step))


def read(k4, v4, step, first, rows, *, count=None, dtype=None, out=None):
    """Rows first[b] + t, t < ``rows`` (an int), of each sequence as numbers.

    first (B,) (None: 0). Returns k, v (B, Hkv, rows, D) of type ``dtype`` (default:
    the steps' type; fp32 where they are bf16), or fills ``out`` = (k, v), whose rows
    are contiguous with strides of whole 16 bytes. Rows outside the cache and, in a
    padded batch, those with t >= count[b] are zeros. Nothing is rounded."""
    rows = int(rows)
    if rows < 0:
        raise ValueError("fbsa.cache4.read: rows must not be negative")
    if dtype is None:
        dtype = out[0].dtype if out is not None else step.dtype
    k, v = (None, None) if out is None else out
    if (k is None) != (v is None):
        raise ValueError("fbsa.cache4.read: out must be (k, v)")
    p = _plan("cache4.read", _plan_rows, (rows, dtype), (k4, v4, step, k, v, first, count))
    if k is None:
        k, v = torch.empty(p.shape, dtype=dtype, device=p.device), torch.empty(p.shape, dtype=dtype, device=p.device)
    if p.empty:
        return (k.zero_(), v.zero_())
    at = (k4.data_ptr(), v4.data_ptr(), step.data_ptr(), k.data_ptr(), v.data_ptr())
    _aligned("cache4.read", at[0] | at[1] | at[3] | at[4])
    if out is not None:
        spans = tuple(zip(at, p.bytes))
        _apart("cache4.read", spans[3:], spans[:3])
    first, count = _int32(first), _int32(count)
    _launch(p, _lib.load().fbsa_cache4_read, "fbsa_cache4_read", *at[:3], _ptr(first), _ptr(count), *at[3:])
    if out is not None:
        increment_version(out)
    return k, v


def _plan_attend(what, scalars, q, k4, v4, step, lens, count, out_gate):
    scale, = scalars
    if q.dim() != 4:
        raise ValueError(f"fbsa.{what}: q must be 4-D")
    B, Hq, T, D = q.shape
    p, d = _Plan(), _lib.Attn4Desc()
    d.dtype = _dtype_code(q)
    held = _held(what, d, k4, v4, step, q.dtype)
    if held[0] != B or held[3] != D:
        raise ValueError(f"fbsa.{what}: q {tuple(q.shape)} does not go with a cache of {held[0]} sequences and head dim {held[3]}")
    if out_gate is not None:
        if out_gate.shape != q.shape or out_gate.dtype != q.dtype:
            raise ValueError(f"fbsa.{what}: out_gate must match q's shape and dtype")
        p.gate_ok = out_gate.stride(-1) == 1
        d.sog[:] = _strides(out_gate, 3) if p.gate_ok else (Hq * T * D, T * D, D)
    _ints(what, "lens", lens, B)
    _ints(what, "count", count, B)
    p.q_ok = _strided(q, 3)
    p.empty = q.numel() == 0
    p.shape, p.S = (B, Hq, T, D), held[2]
    packed = (Hq * T * D, T * D, D)
    d.B, d.Hq, d.Hkv, d.T, d.S, d.D = B, Hq, held[1], T, held[2], D
    d.scale = D ** -0.5 if scale is None else scale
    d.sq[:] = _strides(q, 3) if p.q_ok else packed
    d.so[:] = packed
    p.d = d
    p.nbytes = 0 if p.empty else _lib.load().fbsa_cache4_attn_workspace_bytes(d)
    if p.nbytes == 0 and not p.empty:
        _lib.check(_lib.EINVAL, f"fbsa_cache4_attn ({what})")
    return p


def cache_attention(q, k4, v4, step, lens=None, *, count=None, scale=None, out_gate=None, need_lse=False):
    """Attention of each sequence's newest tokens over its 4-bit cache: the values of
    ``read``, queries, lengths, counts and results as in ``cache.cache_attention``.

    q (B, Hq, T, D) of the rows' type; lens (B,) rows per sequence, the new tokens'
    own among them (default: S). Returns o (B, Hq, T, D), and with need_lse the fp32
    natural-log normaliser (B, Hq, T); padding queries, and queries that see no row,
    give 0 and -inf. A row held as NaN makes the queries that see it NaN, no others.
    """
    what = "cache4.cache_attention"
    scale = None if scale is None else float(scale)
    p = _plan(what, _plan_attend, (scale,), (q, k4, v4, step, lens, count, out_gate))
    o = torch.empty(p.shape, dtype=q.dtype, device=p.device)
    lse = torch.empty(p.shape[:3], dtype=torch.float32, device=p.device) if need_lse else None
    if p.empty:
        return (o, lse) if need_lse else o
    if q.data_ptr() & 15 or not p.q_ok:
        q = q.clone(memory_format=torch.contiguous_format)
        if p.q_ok:  # (the plan describes the tensor that was given)
            return cache_attention(q, k4, v4, step, lens, count=count, scale=scale, out_gate=out_gate, need_lse=need_lse)
    if out_gate is not None and not p.gate_ok:
        out_gate = out_gate.clone(memory_format=torch.contiguous_format)
    pk, pv = k4.data_ptr(), v4.data_ptr()
    _aligned(what, pk | pv)
    lens = torch.full(p.shape[:1], p.S, dtype=torch.int32, device=p.device) if lens is None else _int32(lens)
    count = _int32(count)
    # (256 bytes: the call joins no parts and touches no workspace, so any address does)
    ws = o if p.nbytes == 256 else torch.empty(p.nbytes, dtype=torch.uint8, device=p.device)
    _launch(p, _lib.load().fbsa_cache4_attn, what, q.data_ptr(), pk, pv, step.data_ptr(), lens.data_ptr(), _ptr(count), _ptr(out_gate),
            o.data_ptr(), _ptr(lse), ws.data_ptr(), p.nbytes)
    return (o, lse) if need_lse else o


class KVCache4:
    """One layer's 4-bit cache of B sequences and the calls of a decode loop over it.

    Buffers k4, v4, step (``empty``) and lens (B,) int32 are the object's; all calls
    stay on the device. The caller keeps every sequence within S rows: rows past the
    capacity are dropped by ``append``.
    """

    def __init__(self, B, Hkv, S, D, *, dtype=torch.bfloat16, device="cuda"):
        self.k4, self.v4, self.step = empty(B, Hkv, S, D, dtype=dtype, device=device)
        self.lens = torch.zeros(B, dtype=torch.int32, device=device)
        self.dtype = dtype

    def append(self, k_new, v_new, count=None):
        """New rows (B, Hkv, T, D) behind every sequence (count[b] of them in a padded batch)."""
        append(self.k4, self.v4, self.step, k_new, v_new, self.lens, count=count)
        grow = k_new.shape[2] if count is None else count.clamp(0, k_new.shape[2])
        self.lens.add_(grow).clamp_(max=self.k4.shape[2])

    def attend(self, q, *, count=None, scale=None, out_gate=None, need_lse=False):
        """Attention of the rows just appended."""
        return cache_attention(q, self.k4, self.v4, self.step, self.lens, count=count, scale=scale, out_gate=out_gate, need_lse=need_lse)

    def read(self, rows, *, first=None, count=None, out=None):
        """Rows first[b] + t (default: from the start), t < rows, as numbers of the cache's type (``read``)."""
        return read(self.k4, self.v4, self.step, first, rows, count=count, dtype=self.dtype, out=out)
