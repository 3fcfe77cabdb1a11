"""What the operators of a 4-bit cache refuse, on the host: nothing here launches."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw

from fbsa_amd import _lib, cache4

DUMMY = 1 << 20  # never dereferenced: validation fails first


def _set(d, kw):
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return d


def _rows(**kw):
    d = _lib.Rows4Desc()
    d.dtype, d.B, d.H, d.T, d.S, d.D = _lib.BF16, 2, 2, 3, 128, 64
    d.sk4[:] = d.sv4[:] = (2 * 128 * 32, 128 * 32, 32)
    d.ss[:] = (2 * 128 * 2, 128 * 2)
    d.sk[:] = d.sv[:] = (2 * 3 * 64, 3 * 64, 64)
    return _set(d, kw)


def _attn(**kw):
    d = _lib.Attn4Desc()
    d.dtype, d.B, d.Hq, d.Hkv, d.T, d.S, d.D, d.scale = _lib.BF16, 2, 4, 2, 1, 128, 64, 0.125
    d.sq[:] = d.so[:] = d.sog[:] = (256, 64, 64)
    d.sk4[:] = d.sv4[:] = (2 * 128 * 32, 128 * 32, 32)
    d.ss[:] = (2 * 128 * 2, 128 * 2)
    return _set(d, kw)


def _call(d, ws=DUMMY, nbytes=1 << 40, q=DUMMY, k4=DUMMY, step=DUMMY, lens=DUMMY, gate=None):
    return _lib.load().fbsa_cache4_attn(d, q, k4, DUMMY, step, lens, None, gate, DUMMY, None, ws, nbytes, None)


def test_struct_layouts():
    assert ctypes.sizeof(_lib.Rows4Desc) == 8 + 5 * 8 + 14 * 8
    assert ctypes.sizeof(_lib.Attn4Desc) == 8 + 6 * 8 + 8 + 17 * 8


@pytest.mark.parametrize("kw,needle", [
    ({"dtype": 5}, "dtype"), ({"flags": 1}, "flags"), ({"T": 0}, "positive"), ({"S": 0}, "positive"), ({"B": 0}, "positive"),
    ({"Hkv": 3}, "multiple"), ({"D": 48}, "head dim"), ({"D": 288}, "head dim"), ({"D": 0}, "head dim"), ({"scale": float("nan")}, "scale"),
    ({"scale": 3e38}, "scale"), ({"S": 1 << 31}, "32-bit"), ({"B": 40000}, "grid"), ({"sk4": (8192, 4096, 40)}, "multiples of 16"),
    ({"sv4": (8192, -4096, 32)}, "multiples of 16"), ({"sk4": (0, 0, 1 << 26)}, "64 MiB"), ({"ss": (512, 257)}, "even"), ({"ss": (-2, 256)}, "even"),
    ({"sq": (256, 60, 64)}, "q and o"), ({"so": (256, 64, -64)}, "q and o"), ({"B": 64, "T": 1 << 19}, "grid"),
])
def test_attention_descriptor(kw, needle):
    lib = _lib.load()
    assert lib.fbsa_cache4_attn_workspace_bytes(_attn(**kw)) == 0
    assert needle in lib.fbsa_last_error().decode()
    assert _call(_attn(**kw)) in (_lib.EINVAL, _lib.EUNSUPPORTED)


def test_attention_pointers_and_workspace():
    lib = _lib.load()
    for d in (_attn(), _attn(S=40, T=300)):  # one share: no parts, and still not 0
        need = lib.fbsa_cache4_attn_workspace_bytes(d)
        assert need > 0
        for kw in ({"q": None}, {"k4": None}, {"step": None}, {"lens": None}):
            assert _call(d, **kw) == _lib.EINVAL and b"null" in lib.fbsa_last_error()
        for kw in ({"q": DUMMY + 8}, {"k4": DUMMY + 8}, {"step": DUMMY + 2}, {"lens": DUMMY + 2}, {"gate": DUMMY + 1}):
            assert _call(d, **kw) == _lib.EINVAL and b"aligned" in lib.fbsa_last_error()
        assert _call(d, ws=None) == _lib.EWORKSPACE and _call(d, nbytes=need - 1) == _lib.EWORKSPACE
        assert _call(d, ws=DUMMY + 128, nbytes=need) == _lib.EINVAL
    assert lib.fbsa_cache4_attn_workspace_bytes(None) == 0 and _call(None) == _lib.EINVAL


@pytest.mark.parametrize("kw,needle", [
    ({"dtype": -1}, "dtype"), ({"flags": 2}, "flags"), ({"T": 0}, "positive"), ({"H": 0}, "positive"), ({"D": 8}, "head dim"),
    ({"D": 320}, "head dim"), ({"S": 1 << 31}, "32-bit"), ({"H": 70000}, "grid"), ({"B": 1 << 14, "H": 8}, "grid"),
    ({"sk4": (8192, 4096, 8)}, "multiples of 16"), ({"sv4": (-16, 4096, 32)}, "multiples of 16"), ({"ss": (511, 256)}, "even"),
    ({"sk": (384, 192, 60)}, "rows"), ({"sv": (384, -192, 64)}, "rows"), ({"dtype": _lib.F32, "sk": (384, 192, 66)}, "rows"),
    ({"B": 64, "H": 64, "T": 1 << 15}, "grid"),
])
def test_rows_descriptor(kw, needle):
    lib = _lib.load()
    for fn in (lib.fbsa_cache4_append, lib.fbsa_cache4_read):
        assert fn(_rows(**kw), DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, None, None) in (_lib.EINVAL, _lib.EUNSUPPORTED)
        assert needle in lib.fbsa_last_error().decode()


def test_rows_pointers():
    lib = _lib.load()
    for fn, order in ((lib.fbsa_cache4_append, (0, 1, 2, 3, 4)), (lib.fbsa_cache4_read, (0, 1, 2, 5, 6))):
        assert fn(None, *[DUMMY] * 7, None) == _lib.EINVAL
        for i in order:
            args = [DUMMY] * 7
            args[i] = None
            assert fn(_rows(), *args, None) == _lib.EINVAL and b"null" in lib.fbsa_last_error()
            args[i] = DUMMY + 2
            assert fn(_rows(), *args, None) == _lib.EINVAL and b"aligned" in lib.fbsa_last_error()
    args = [DUMMY] * 7
    args[5] = None  # an append without places
    assert lib.fbsa_cache4_append(_rows(), *args, None) == _lib.EINVAL


def test_what_the_python_side_refuses():
    k4, v4, step = cache4.empty(2, 2, 30, 64, device="cpu")
    x = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    q, lens = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    calls = [
        (lambda: cache4.cache_attention(q, k4, v4, step, lens), "no CPU path"),
        (lambda: cache4.append(k4, v4, step, x, x, lens), "no CPU path"),
        (lambda: cache4.read(k4, v4, step, lens, 3), "no CPU path"),
        (lambda: cache4.read(k4, v4, step, lens, -1), "negative"),
        (lambda: cache4.read(k4, v4, step, lens, 3, out=(x, None)), "out must be"),
        (lambda: cache4.append(k4, v4, step, x[0], x[0], lens), "4-D"),
        (lambda: cache4.append(k4, v4, step, x, x, None), "required"),
        (lambda: cache4.cache_attention(q.clone().requires_grad_(), k4, v4, step, lens), "gradients"),
        (lambda: cache4.empty(1, 1, 8, 40, device="cpu"), "head dim"),
        (lambda: cache4.empty(1, 1, 8, 288, device="cpu"), "head dim"),
    ]
    for i, (call, text) in enumerate(calls):
        with pytest.raises(ValueError, match=text):
            call()
            raise AssertionError(f"call {i} was accepted")
    with fw.dual_level(), torch.no_grad(), pytest.raises(ValueError, match="gradients"):
        cache4.cache_attention(fw.make_dual(q, torch.ones_like(q)), k4, v4, step, lens)
