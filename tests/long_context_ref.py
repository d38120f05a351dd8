"""Plain 64-bit forms of the operators for long contexts, and bounds of what 16-bit operands and results may be off.

A rounding to a type is off by at most half a step, u = eps / 2 of the type, relative to the value (2^-25 absolute where
fp16 has no smaller steps).  Sums in 32 bits add a few times 2^-24 of the sum of absolute values; SLACK stands for them, for
the exponential's 2^-22 and for products of bounds.
"""
import math

import torch

SLACK = 2e-5


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def visible(q_len, kv_len, window, sinks, length, device):
    p = torch.arange(q_len, device=device)[:, None] + kv_len - q_len
    j = torch.arange(kv_len, device=device)[None]
    seen = j <= p
    if window > 0:
        seen &= (j > p - window) | (j < sinks)
    return seen & (p < length) & (j < length)


def window_attention(q, k, v, window, sinks, lengths, scale, dout=None):
    """out, lse and, with dout, dq, dk, dv in 64 bits, each with its bound; rows that are not there hold NaN in the values."""
    u = unit(q.dtype)
    B, Tq, H, d = q.shape
    Tk, G = k.shape[1], H // k.shape[2]
    q, k, v = (x.double() for x in (q, k, v))
    r = {n: torch.full(s, math.nan, dtype=torch.float64, device=q.device)
         for n, s in (("out", q.shape), ("lse", (B, H, Tq)), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    e = {n: torch.zeros_like(t) for n, t in r.items()}
    for b in range(B):
        n = Tk if lengths is None else int(lengths[b])
        rows = max(0, n - (Tk - Tq))
        if n <= 0:
            continue
        seen = visible(Tq, Tk, window, sinks, n, q.device)[:rows, :n]
        if dout is not None:
            r["dk"][b, :n] = r["dv"][b, :n] = 0
        if rows <= 0:
            continue
        for h in range(H):
            qh, kh, vh = q[b, :rows, h], k[b, :n, h // G], v[b, :n, h // G]
            s = qh @ kh.T * scale
            size = (qh.abs() @ kh.abs().T * abs(scale)).masked_fill(~seen, 0).amax(-1, keepdim=True) + 1  # what the scores' sums are made of
            s = s.masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(s, -1, keepdim=True)
            p = torch.exp(s - lse)
            o = p @ vh
            off = SLACK * size                      # of a weight, relative
            weighted = p @ vh.abs()
            r["out"][b, :rows, h], r["lse"][b, h, :rows] = o, lse[:, 0]
            tiny = 2.0 ** -24 * (seen.double() @ vh.abs())   # weights below fp16's smallest steps
            e["out"][b, :rows, h] = (u + 2 * off) * weighted + u * o.abs() + tiny + 2.0 ** -25
            e["lse"][b, h, :rows] = SLACK * (size[:, 0] + lse[:, 0].abs())
            if dout is None:
                continue
            g = dout[b, :rows, h].double()
            dp = g @ vh.T
            D = (g * o).sum(-1, keepdim=True)
            ds = p * (dp - D) * scale
            eo = e["out"][b, :rows, h] + u * o.abs()         # the output that the backward pass is given
            eD = (g.abs() * eo).sum(-1, keepdim=True) + SLACK * (g.abs() * o.abs()).sum(-1, keepdim=True)
            eds = abs(scale) * p * (eD + SLACK * (g.abs() @ vh.abs().T)) + ds.abs() * (u + 2 * off) + 2.0 ** -24 * seen
            r["dq"][b, :rows, h] = ds @ kh
            e["dq"][b, :rows, h] = eds @ kh.abs() + SLACK * (ds.abs() @ kh.abs())
            r["dk"][b, :n, h // G] += ds.T @ qh
            e["dk"][b, :n, h // G] += eds.T @ qh.abs() + SLACK * (ds.abs().T @ qh.abs())
            r["dv"][b, :n, h // G] += p.T @ g
            e["dv"][b, :n, h // G] += (p * (u + 2 * off) + 2.0 ** -24 * seen).T @ g.abs()
    for n in ("dq", "dk", "dv"):
        e[n] += u * r[n].nan_to_num().abs() + 2.0 ** -25
    return r, e


def worst(got, want, bound):
    """The largest error as a share of its bound, over the values that there are."""
    there = ~want.isnan()
    if not there.any():
        return 0.0
    return float(((got.double() - want).abs() / bound)[there].nan_to_num(nan=math.inf).max())
