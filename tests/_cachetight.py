"""Attention over a cache in 64 bits with what its tight error bounds need:
sum p |v| of every output, and infinite keys and values as the formulas have them."""
import math

import torch

from _cacheref import HALF


def attend(q, k, v, lens, count=None, kp=None, vp=None, scale=None, gate=None, weight=None):
    """dict of o, lse, w (or None), and per output: a = sum p |v|, a2 = sum p^2 v^2
    (both times the gate), v1 = sum |v| over the rows seen; big = the largest
    sum |q_d k_d| |scale|. A key scored -inf drops out, with its value; a row of
    which every key did, or that sees none, has o = 0 and lse = -inf."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    B, Hq, T, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    shape = (B, Hq, T, D)
    r = {x: torch.zeros(shape, dtype=torch.float64) for x in ("o", "a", "a2", "v1")}
    r["lse"] = torch.full(shape[:3], -math.inf, dtype=torch.float64)
    r["w"] = None if weight is None else weight.detach().cpu().double().clone()
    r["big"] = 0.0
    P = 0 if kp is None else kp.shape[1]
    if P:
        kp, vp = kp.detach().cpu().double(), vp.detach().cpu().double()
    for b in range(B):
        n = min(max(int(lens[b]), 0), S)
        c = T if count is None else min(max(int(count[b]), 0), T)
        place = P + n - c + torch.arange(c).view(c, 1)   # the last row that each query sees
        for h in range(Hkv):
            kb, vb = k[b, h, :n], v[b, h, :n]
            if P:
                kb, vb = torch.cat([kp[h], kb]), torch.cat([vp[h], vb])
            seen = (torch.arange(P + n) <= place) | (torch.arange(P + n) < P)
            bad = ~vb.isfinite()
            fin = vb.masked_fill(bad, 0.0)
            for hq in range(h * G, h * G + G):
                if not c or not P + n:
                    continue
                qq = q[b, hq, :c]
                x = (qq @ kb.t() * scale).masked_fill(~seen, -math.inf)
                mag = (qq.abs() @ kb.abs().t()).masked_fill(~seen, 0.0)
                r["big"] = max(r["big"], float(mag.masked_fill(mag.isinf(), 0.0).max()) * abs(scale))
                lse = x.logsumexp(-1)
                some = ~(lse == -math.inf).view(c, 1)
                p = (x - lse.masked_fill(lse == -math.inf, 0.0).view(c, 1)).exp() * some
                r["lse"][b, hq, :c] = lse
                o = p @ fin
                for s in bad.any(1).nonzero().flatten().tolist():   # (0 * inf only where the key is seen and has p > 0)
                    term = torch.where(bad[s], vb[s], 0.0).expand(c, D)
                    o = torch.where((x[:, s] > -math.inf).view(c, 1) & bad[s], o + p[:, s:s + 1] * term, o)
                r["o"][b, hq, :c] = o
                r["a"][b, hq, :c] = p @ fin.abs()
                r["a2"][b, hq, :c] = p.square() @ fin.square()
                r["v1"][b, hq, :c] = seen.double() @ fin.abs()
                if r["w"] is not None:
                    r["w"][b, h, :n] += p[:, P:].sum(0)
    if gate is not None:
        s = gate.detach().cpu().double().sigmoid()
        for x, y in (("o", s), ("a", s), ("a2", s * s), ("v1", s)):
            r[x] = r[x] * y
    return r


def check(got, r, q, keys, rounded, gate=False):
    """o, lse, w against attend's, element by element, and o's relative L2 error.

    keys: how many a row may see. A probability's relative error e: the score is
    a D-term fp32 sum of terms up to `big` in the natural exponent, then scaled,
    shifted and exponentiated, (D + 4) steps of 2^-24 of big and 2^-20 for the
    instructions; the row sum adds a step per key, twice where parts are joined.
    o = sum p v is then off by 2 e sum p |v| (its own sum and the row's), by P's
    rounding: half a step h of each p where it is rounded once (`rounded`), 2^-16
    where it goes as a pair, and fp16's smallest parts, 2^-25 of sum |v| as the
    row's sum is at least 1; the gate's sigmoid 2^-21 of o; o's storage h of o, or half a
    subnormal step (fp16 numbers below 2^-14 are 2^-24 apart).
    The roundings of P and o are independent and unbiased, each at most h of its
    term, so of standard deviation at most h / sqrt(3): the L2 error stays below
    1.25 sqrt(h^2 / 3 (sum o^2 + sum p^2 v^2)) and the small terms' bound."""
    o, lse, w = got
    D, h = q.shape[-1], HALF[q.dtype]
    half = q.dtype != torch.float32
    o, lse = o.cpu().double(), lse.cpu().double()
    e = (D + 4) * 2.0 ** -24 * r["big"] + 2.0 ** -20 + 2 * keys * 2.0 ** -24
    small = 2 * e * r["a"] + (2.0 ** -25 * r["v1"] if q.dtype == torch.float16 else 0.0)
    if half and not rounded:
        small = small + 2.0 ** -16 * r["a"]
    if gate:
        small = small + 2.0 ** -21 * r["o"].abs().nan_to_num(0.0, 0.0, 0.0)
    bound = small + (h * r["a"] if half and rounded else 0.0)
    ro, rl = r["o"], r["lse"]
    fin = ro.isfinite()
    assert torch.equal(o.isnan(), ro.isnan()) and torch.equal(o[ro.isinf()], ro[ro.isinf()]) and o[fin].isfinite().all()
    err = (o - ro).abs()[fin]
    tiny = torch.finfo(q.dtype).smallest_normal * h   # half a step below the smallest normal number (fp16: 2^-25)
    excess = (err - (h + 2.0 ** -30) * ro.abs()[fin] - bound[fin] - tiny)
    assert not len(excess) or excess.max() <= 0, f"o off by {float(excess.max()):.3e} more than its bound"
    if half and fin.sum() >= 4096:
        var = h * h / 3 * (ro[fin].square().sum() + (r["a2"][fin].sum() if rounded else 0.0))
        l2, most = err.square().sum().sqrt(), 1.25 * var.sqrt() + small[fin].square().sum().sqrt()
        assert l2 <= most, f"o's L2 error {float(l2):.3e}, bound {float(most):.3e}"
    assert torch.equal(lse.isnan(), rl.isnan()) and torch.equal(lse.isinf(), rl.isinf())
    fin = rl.isfinite()
    if fin.any():
        assert ((lse - rl)[fin].abs() - 2.0 ** -23 * rl[fin].abs()).max() <= e
    if w is not None:
        w, rw, rows = w.cpu().double(), r["w"], q.shape[1] * q.shape[2]
        assert torch.equal(w.isnan(), rw.isnan())
        fin = ~rw.isnan()
        assert ((w - rw)[fin].abs() - (2 * e + (rows + 1) * 2.0 ** -24) * rw[fin].abs()).max() <= 1e-30
