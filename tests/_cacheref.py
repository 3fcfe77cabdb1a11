"""Plain 64-bit forms of the cache operators, on the CPU, and the error bounds
that their GPU kernels' arithmetic admits."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step of the output


def attend(q, k, v, lens, count=None, kp=None, vp=None, scale=None, gate=None, weight=None):
    """(o, lse, out_weight or None, score bound): lists over sequences, one softmax
    over the prefix and the visible rows; rows at or past lens are not looked at."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    B, Hq, T, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    o = torch.zeros(B, Hq, T, D, dtype=torch.float64)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64)
    w = None if weight is None else weight.detach().cpu().double().clone()
    big = 0.0
    P = 0 if kp is None else kp.shape[1]
    for b in range(B):
        n = min(max(int(lens[b]), 0), S)
        c = T if count is None else min(max(int(count[b]), 0), T)
        for h in range(Hq):
            kb, vb = k[b, h // G, :n], v[b, h // G, :n]
            if P:
                kb = torch.cat([kp.detach().cpu().double()[h // G], kb])
                vb = torch.cat([vp.detach().cpu().double()[h // G], vb])
            for t in range(c):
                m = P + min(max(n - c + t + 1, 0), n)
                if m == 0:
                    continue
                x = kb[:m] @ q[b, h, t] * scale
                big = max(big, float((kb[:m].abs() @ q[b, h, t].abs()).max()) * abs(scale))
                lse[b, h, t] = x.logsumexp(0)
                p = (x - lse[b, h, t]).exp()
                o[b, h, t] = p @ vb[:m]
                if w is not None and m > P:
                    w[b, h // G, :m - P] += p[P:]
    if gate is not None:
        o = o * gate.detach().cpu().double().sigmoid()
    return o, lse, w, big


def bounds(q, v, S, big, rounded):
    """Absolute error bounds (o beyond its storage rounding as a multiple of |v|,
    lse, relative error of a probability).

    A score is a D-term fp32 sum, its scaling and the exponent's argument: at
    most (D + 4) steps of 2^-24 of its absolute terms (`big`) in the natural
    exponent, and the exponential and log2 instructions one or two units in the
    last place: 2^-22. A row's sum over S keys adds at most S 2^-24 relative,
    its parts joined with two more exponentials. A probability in the value
    product is a pair of 16-bit numbers: for bf16 cut at 2^-7 and the rest
    rounded at 2^-9 of itself (2^-16 relative), for fp16 better than that, or
    2^-25 absolute where the rest is subnormal, at most S of them against a row
    sum of at least 1; fp32 none. Where many rows share their keys (`rounded`)
    it is rounded once to the operand type: each is off by at most half a step
    of itself, so sum p v by at most half a step of sum p |v| (and, for fp16,
    2^-25 for each subnormal one)."""
    D = q.shape[-1]
    score = (D + 4) * 2.0 ** -24 * big + 2.0 ** -22 * 4
    total = score + S * 2.0 ** -24
    split = 0.0 if q.dtype == torch.float32 else (HALF[q.dtype] if rounded else 2.0 ** -16) + S * 2.0 ** -25
    return 2 * total + split, total + 2.0 ** -22, 2 * total


def many_rows(q, Hkv, P=0):
    """Whether the rows of a (sequence, KV head), or those that share a prefix,
    are more than one 16-row tile."""
    rows = q.shape[2] * (q.shape[1] // Hkv)
    return rows > 16 or (P > 0 and q.shape[0] * rows > 16)


def check_attend(got, ref, q, v, S, rounded):
    o, lse, w = got
    ro, rl, rw, big = ref
    tol_o, tol_l, tol_p = bounds(q, v, S, big, rounded)
    o, lse = o.cpu().double(), lse.cpu().double()
    vmax = max(1.0, float(v.detach().abs().nan_to_num(0.0).max()))
    excess = ((o - ro).abs() - HALF[q.dtype] * ro.abs() - tol_o * vmax).max()
    assert not torch.isnan(o).any() and excess <= 0, f"o off by {excess:.3e} more than {tol_o * vmax:.3e} and its rounding"
    assert torch.equal(lse.isinf(), rl.isinf())
    fin = ~rl.isinf()
    if fin.any():
        err = ((lse - rl)[fin].abs() - 2.0 ** -23 * rl[fin].abs()).max()
        assert err <= tol_l, f"lse off by {err:.3e}, bound {tol_l:.3e}"
    if w is not None:
        # (each of the group's queries adds one rounding; what was there before, one)
        rows = q.shape[1] * q.shape[2]
        w = w.cpu().double()
        err = ((w - rw).abs() - (tol_p + (rows + 1) * 2.0 ** -24) * rw.abs()).max()
        assert not torch.isnan(w).any() and err <= 1e-30, f"weight off by {err:.3e}"


def evict(k, v, w, lens, budget, recent, sink):
    """Per (sequence, head) lists of kept rows."""
    B, H, S, _ = k.shape
    keep = []
    for b in range(B):
        n = min(max(int(lens[b]), 0), S)
        for h in range(H):
            rows = list(range(n))
            if n > budget:
                x = w[b, h, sink:n - recent].tolist()
                x = [-math.inf if math.isnan(y) else y for y in x]
                best = sorted(range(len(x)), key=lambda i: (-x[i], i))[:budget - sink - recent]
                rows = list(range(sink)) + sorted(i + sink for i in best) + list(range(n - recent, n))
            keep.append(rows)
    return keep
