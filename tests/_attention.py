"""The attention operators from their definitions in 64 bits (on the host), with
an elementwise bound of the error that a 16-bit kernel may make.

The bounds count, for a storage type whose rounding is off by at most half a
step u (2^-11 f16, 2^-8 bf16) relative to the value:
  - the output's own rounding, u |out|;
  - the rounding of each probability P (and of dS) to that type, u per term, and
    in f16 half the smallest step, 2^-25 in the scale the term is held in;
  - the f32 arithmetic behind each term: a sum of n products is off by at most
    n 2^-24 of the sum of their magnitudes, an exponential by 2^-22 of its value
    plus the error of its argument.
"""
from __future__ import annotations

import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E32 = 2.0 ** -24


def segments(rows, nbatch, offsets):
    if offsets is not None:
        return [(offsets[b], offsets[b + 1]) for b in range(nbatch)]
    n = rows // nbatch
    return [(b * n, (b + 1) * n) for b in range(nbatch)]


def _pairs(q, k, nbatch, q_offsets, k_offsets, k_lens):
    for b, ((q0, q1), (k0, k1)) in enumerate(zip(segments(q.shape[0], nbatch, q_offsets),
                                                 segments(k.shape[0], nbatch, k_offsets))):
        n = k1 - k0 if k_lens is None else min(k1 - k0, max(k_lens[b], 0))
        yield slice(q0, q1), slice(k0, k0 + n)


def _f64(t):
    return t.detach().cpu().double()


def forward(q, k, v, scale, nbatch=1, q_offsets=None, k_offsets=None, k_lens=None):
    """(out, lse, bound of out, bound of lse), float64; rows outside the segments are NaN."""
    u = U[q.dtype]
    f16 = q.dtype == torch.float16
    q, k, v = _f64(q), _f64(k), _f64(v)
    t, h, d = q.shape
    g = h // k.shape[1]
    out = torch.full((t, h, d), math.nan, dtype=torch.float64)
    lse = torch.full((h, t), math.nan, dtype=torch.float64)
    bo, bl = torch.zeros_like(out), torch.zeros_like(lse)
    for qr, kr in _pairs(q, k, nbatch, q_offsets, k_offsets, k_lens):
        for i in range(h):
            qi, ki, vi = q[qr, i], k[kr, i // g], v[kr, i // g]
            n = ki.shape[0]
            if n == 0:
                out[qr, i] = 0.0
                lse[i, qr] = -math.inf
                continue
            s = qi @ ki.t() * scale
            lse[i, qr] = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[i, qr][:, None])
            out[qr, i] = p @ vi
            es = scale * (d + 8) * E32 * (qi.abs() @ ki.abs().t()) + 4 * E32 * s.abs() + 2.0 ** -22
            ep = es + es.amax(1, keepdim=True) + n * E32        # numerator and sum
            bo[qr, i] = u * out[qr, i].abs() + (p * (u + 2 * ep + n * E32)) @ vi.abs()
            if f16:
                bo[qr, i] += 2.0 ** -25 * vi.abs().sum(0) + 2.0 ** -25
            bl[i, qr] = es.amax(1) + n * E32 + 4 * E32 * lse[i, qr].abs() + 2.0 ** -22
    return out, lse, bo, bl


def backward(dout, q, k, v, out, lse, scale, nbatch=1, q_offsets=None, k_offsets=None, k_lens=None):
    """[(dq, bound), (dk, bound), (dv, bound)], float64, from the given out and lse."""
    u = U[q.dtype]
    f16 = q.dtype == torch.float16
    dout, q, k, v, out, lse = (_f64(t) for t in (dout, q, k, v, out, lse))
    t, h, d = q.shape
    g = h // k.shape[1]
    dq, bq = torch.full_like(q, math.nan), torch.zeros_like(q)
    dk, dv, bk, bv = (torch.zeros_like(k) for _ in range(4))
    for x, (k0, k1) in zip(range(nbatch), segments(k.shape[0], nbatch, k_offsets)):
        del x
    covered = torch.zeros(k.shape[0], dtype=torch.bool)
    for k0, k1 in segments(k.shape[0], nbatch, k_offsets):
        covered[k0:k1] = True
    dk[~covered] = math.nan
    dv[~covered] = math.nan
    for qr, kr in _pairs(q, k, nbatch, q_offsets, k_offsets, k_lens):
        for i in range(h):
            j = i // g
            qi, ki, vi, go = q[qr, i], k[kr, j], v[kr, j], dout[qr, i]
            n, m = ki.shape[0], qi.shape[0]
            if n == 0 or m == 0:
                dq[qr, i] = 0.0
                continue
            s = qi @ ki.t() * scale
            p = torch.exp(s - lse[i, qr][:, None])
            delta = (go * out[qr, i]).sum(1, keepdim=True)
            dp = go @ vi.t()
            ds = p * (dp - delta)
            es = scale * (d + 8) * E32 * (qi.abs() @ ki.abs().t()) + 4 * E32 * (s.abs() + lse[i, qr].abs()[:, None]) \
                + 2.0 ** -22
            inner = (d + 4) * E32 * (go.abs() @ vi.abs().t() + (go.abs() * out[qr, i].abs()).sum(1, keepdim=True))
            eds = ds.abs() * (u + 2 * es) + p * inner * (1 + u)
            if f16:
                eds += 2.0 ** -37 * go.norm(dim=1).amax() * vi.norm(dim=1).amax()
            dq[qr, i] = scale * (ds @ ki)
            bq[qr, i] = u * dq[qr, i].abs() + scale * ((eds + n * E32 * ds.abs()) @ ki.abs())
            epv = p * (u + 2 * es + m * g * E32) + (2.0 ** -39 if f16 else 0.0)
            dv[kr, j] += p.t() @ go
            bv[kr, j] += epv.t() @ go.abs()
            dk[kr, j] += scale * (ds.t() @ qi)
            bk[kr, j] += scale * ((eds + m * g * E32 * ds.abs()).t() @ qi.abs())
    bk += u * dk.abs().nan_to_num()
    bv += u * dv.abs().nan_to_num()
    if f16:
        for b in (bq, bk, bv):
            b += 2.0 ** -25
    return [(dq, bq), (dk, bk), (dv, bv)]


def check(got, want, bound, what):
    """got within bound of want where want is finite, equal to it where infinite."""
    got = _f64(got)
    live = torch.isfinite(want)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities"
    err = (got - want).abs()[live]
    assert torch.isfinite(got[live]).all(), f"{what}: non-finite values"
    over = err > bound[live]
    assert not over.any(), f"{what}: {int(over.sum())} of {over.numel()} past the bound, worst " \
                           f"{float((err / bound[live].clamp_min(1e-300)).max()):.3f} of it"
