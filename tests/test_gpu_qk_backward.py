"""The q/k epilogue's gradients against their definition in 64 bits.

Bounds, per element: u |dx| for the storage rounding (u half a step: 2^-24 f32,
2^-11 f16, 2^-8 bf16), and f32 arithmetic of values whose size is w = |g gamma|
sqrt(D): the rotation's two products (2 steps, and 2^-23 of the angle's cos and
sin each), the norm's sum of D squares ((D / 2 + 4) 2^-24 relative: half of a
sum's error passes through the square root) and v_rsq_f32 (2^-22), the dot
product (D 2^-24 of the sum of magnitudes). 1 / n scales it. dgamma and dbias:
the terms' own errors and rows * 2^-24 of the sum of their magnitudes.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
E = 2.0 ** -24


def freqs(d, axes=3):
    n = d // 2 // axes
    return (np.float32(1) / np.float32(10000) ** (np.arange(n, dtype=np.float32) / np.float32(n))).astype(np.float32)


def cos_sin(rows, d, f, pos):
    """float64 cos and sin [rows, D/2] of the f32 angles; pos int [rows, axes] or None."""
    a = np.zeros((rows, d // 2), np.float32)
    if pos is not None:
        ang = pos.astype(np.float32)[:, :, None] * f[None, None, :]
        a[:, :ang.shape[1] * f.size] = ang.reshape(rows, -1)
    a = torch.from_numpy(a).double()
    return a.cos(), a.sin()


def reference(x, dy, gamma, bias, cs, dtype):
    """(dx, its bound, dgamma, its bound, dbias, its bound)."""
    dy = dy.cpu().double()
    rows, h, d = dy.shape
    u = U[dtype]
    c, s = (t[:, None] for t in cs)
    re, im = dy[..., 0::2], dy[..., 1::2]
    g = torch.stack([re * c + im * s, im * c - re * s], -1).reshape(rows, h, d)
    size = (re.abs() + im.abs()).repeat_interleave(2, -1)
    eg = 8 * E * size                                   # rotation: cos, sin and two products
    if gamma is None:
        dx, edx = g, eg
        dg = eg_sum = None
    else:
        x = x.cpu().double()
        if bias is not None:
            x = x + bias.cpu().double()
        gm = gamma.cpu().double()
        n = x.norm(dim=-1, keepdim=True)
        floor = n < 1e-12
        n = n.clamp_min(1e-12)
        xh = x / n
        rel = (d / 2 + 8) * E + 2.0 ** -22              # of xh and 1 / n
        exh = rel * xh.abs() + (E * x.abs() / n if bias is not None else 0)
        w = g * gm * math.sqrt(d)
        ew = eg * gm.abs() * math.sqrt(d) + 3 * E * w.abs()
        dot = (w * xh).sum(-1, keepdim=True)
        edot = (ew * xh.abs() + w.abs() * exh).sum(-1, keepdim=True) + d * E * (w * xh).abs().sum(-1, keepdim=True)
        dot, edot = dot.masked_fill(floor, 0), edot.masked_fill(floor, 0)
        num = w - xh * dot
        dx = num / n
        edx = (ew + exh * dot.abs() + xh.abs() * edot + 2 * E * (xh * dot).abs() + (rel + 2 * E) * num.abs()) / n
        dg = (g * xh).sum(0) * math.sqrt(d)
        eg_sum = ((eg * xh.abs() + g.abs() * exh).sum(0) + rows * E * (g * xh).abs().sum(0)) * math.sqrt(d) + 2 * E * dg.abs()
    db = dx.sum(0)
    edb = edx.sum(0) + rows * E * dx.abs().sum(0)
    return dx, edx + u * dx.abs() + (2.0 ** -25 if dtype == F16 else 0), dg, eg_sum, db, edb


def check(got, want, bound, what):
    got = got.cpu().double()
    assert torch.isfinite(got).all(), what
    bad = (got - want).abs() > bound
    assert not bad.any(), f"{what}: worst {float(((got - want).abs() / bound.clamp_min(1e-300)).max()):.3f} of the bound"


def tensors(seed, rows, h, d, dtype, dev, n=4):
    g = torch.Generator().manual_seed(seed)
    out = [torch.randn((rows, h, d), generator=g).to(dtype).to(dev) for _ in range(n)]
    par = [(torch.randn((h, d), generator=g) * 0.1 + m).to(dev) for m in (1.0, 1.0, 0.0, 0.0)]
    return out, par


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,h,d", [(1, 1, 64), (3, 12, 128), (37, 16, 64), (129, 4, 128), (50, 5, 64), (700, 16, 128),
                                      (20, 20, 128), (33, 3, 96), (9, 2, 256), (11, 7, 2)])
def test_norm_bias_and_coords(dev, dtype, rows, h, d):
    from t2h import ops

    (q, k, dq, dk), (gq, gk, bq, bk) = tensors(rows + d, rows, h, d, dtype, dev)
    f = freqs(d)
    pos = np.random.default_rng(rows).integers(0, 128, (rows, 3)).astype(np.int32)
    coords = torch.from_numpy(np.concatenate([np.zeros((rows, 1), np.int32), pos], 1)).to(dev)
    dqi, dki, dgq, dgk, dbq, dbk = ops.qk_rmsnorm_rope_backward(
        dq=dq, dk=dk, q=q, k=k, gamma_q=gq, gamma_k=gk, bias_q=bq, bias_k=bk, freqs=f, coords=coords)
    cs = cos_sin(rows, d, f, pos)
    for x, dy, gm, bs, got in ((q, dq, gq, bq, (dqi, dgq, dbq)), (k, dk, gk, bk, (dki, dgk, dbk))):
        dx, edx, dg, edg, db, edb = reference(x, dy, gm, bs, cs, dtype)
        check(got[0], dx, edx, "dx")
        check(got[1], dg, edg, "dgamma")
        check(got[2], db, edb, "dbias")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("source", ["none", "grid", "phases"])
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("rows,h", [(150, 4), (47, 9), (128, 3)])
def test_one_tensor_position_sources_and_no_norm(dev, dtype, source, d, rows, h):
    from t2h import ops

    (q, _, dq, _), (gq, _, bq, _) = tensors(d, rows, h, d, dtype, dev)
    f = freqs(d)
    kw, pos = dict(use_rope=False), None
    if source != "none":
        r = 4
        i = np.arange(rows) % r ** 3
        pos = np.stack([i // (r * r), i // r % r, i % r], 1)
        kw = dict(freqs=f, grid_res=r)
        if source == "phases":
            kw = dict(phases=ops.rope_phases(r ** 3, d, f, grid_res=r, device=dev), freqs=f)
    cs = cos_sin(rows, d, f, pos)
    for which in "qk":
        for gm, bs in ((gq, bq), (gq, None), (None, bq), (None, None)):
            r = ops.qk_rmsnorm_rope_backward(**{"d" + which: dq, which: q, "gamma_" + which: gm, "bias_" + which: bs}, **kw)
            dx, edx, dg, edg, db, edb = reference(q, dq, gm, bs, cs, dtype)
            i = "qk".index(which)
            check(r[i], dx, edx, "dx")
            assert r[1 - i] is None and r[3 - i] is None and r[5 - i] is None
            if gm is not None:
                check(r[2 + i], dg, edg, "dgamma")
            if bs is not None:
                check(r[4 + i], db, edb, "dbias")
            else:
                assert r[4 + i] is None


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,h,d", [(211, 12, 128), (40, 13, 64)])
def test_packed_views_and_in_place(dev, dtype, rows, h, d):
    from t2h import ops

    g = torch.Generator().manual_seed(0)
    qkv = torch.randn((rows, 3, h, d), generator=g).to(dtype).to(dev)
    dqkv = torch.randn((rows, 3, h, d), generator=g).to(dtype).to(dev)
    gq, gk = ((torch.randn((h, d), generator=g) * 0.1 + 1).to(dev) for _ in range(2))
    kw = dict(q=qkv[:, 0], k=qkv[:, 1], gamma_q=gq, gamma_k=gk, freqs=freqs(d), grid_res=16)
    want = ops.qk_rmsnorm_rope_backward(dq=dqkv[:, 0], dk=dqkv[:, 1], **kw)
    dv = dqkv[:, 2].clone()
    x = qkv.clone()
    got = ops.qk_rmsnorm_rope_backward(dq=dqkv[:, 0], dk=dqkv[:, 1], in_place=True, **kw)
    assert got[0].data_ptr() == dqkv.data_ptr()
    for a, b in zip(got[:4], want[:4]):
        assert torch.equal(a, b)
    assert torch.equal(dqkv[:, 2], dv) and torch.equal(qkv, x)
    # an odd element offset: the path without vector loads, the same values to rounding
    buf = torch.empty((rows * h * d + 1,), dtype=dtype, device=dev)
    odd = buf[1:].view(rows, h, d).copy_(want[0].float() * 0 + qkv[:, 0])
    r = ops.qk_rmsnorm_rope_backward(dq=odd, q=qkv[:, 0].contiguous(), gamma_q=gq, use_rope=False)
    dx, edx, dg, edg, _, _ = reference(qkv[:, 0], odd, gq, None, cos_sin(rows, d, freqs(d), None), dtype)
    check(r[0], dx, edx, "dx")
    check(r[2], dg, edg, "dgamma")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [128, 96])
def test_rows_of_zero_and_near_it(dev, dtype, d):
    """|x| below 1e-12: n is a constant, dx = w / 1e-12."""
    from t2h import ops

    (q, _, dq, _), (gq, _, _, _) = tensors(5, 8, 2, d, dtype, dev)
    q[1] = 0
    q[2] = 1e-16
    q[3, 1] = 0
    dq[1:3] *= 1e-6
    r = ops.qk_rmsnorm_rope_backward(dq=dq, q=q, gamma_q=gq, use_rope=False)
    dx, edx, dg, edg, _, _ = reference(q, dq, gq, None, cos_sin(8, d, freqs(d), None), dtype)
    check(r[0], dx, edx, "dx")
    check(r[2], dg, edg, "dgamma")


def test_agrees_with_the_forward_by_differences(dev):
    """Central differences of the forward kernel in f32: sum(y * dy) changes by
    dx . direction. The forward's rounding: 2^-21 of each |y|, random over the
    sum, divided by the step; the difference's own error is of order step^2."""
    from t2h import ops

    rows, h, d = 40, 4, 64
    (q, _, dq, _), (gq, _, bq, _) = tensors(9, rows, h, d, F32, dev)
    f = freqs(d)
    kw = dict(freqs=f, grid_res=4)
    dx, _, dg, _, db, _ = ops.qk_rmsnorm_rope_backward(dq=dq, q=q, gamma_q=gq, bias_q=bq, **kw)
    gen = torch.Generator().manual_seed(1)
    for i, grad in enumerate((dx, dg, db)):
        base = [q, gq, bq]
        dirn = torch.randn(base[i].shape, generator=gen).to(dev)
        step = 1e-2
        vals = []
        mags = 0.0
        for sgn in (1, -1):
            y = list(base)
            y[i] = y[i] + sgn * step * dirn
            out = ops.qk_rmsnorm_rope(q=y[0], gamma_q=y[1], bias_q=y[2], **kw)[0].double()
            vals.append((out * dq.double()).sum())
            mags = float((out * dq.double()).pow(2).sum().sqrt())
        want = float(vals[0] - vals[1]) / (2 * step)
        got = float((grad.double() * dirn.double()).sum())
        # third-order term: |x| = 8, a step of 1e-2 turns xh by 1e-2, relative (step / 1)^2 of the gradient's size
        size = float((grad.double() * dirn.double()).pow(2).sum().sqrt())
        assert abs(got - want) <= 2.0 ** -21 * mags / step * 4 + step ** 2 * size * 4 + 1e-6 * abs(want)


def test_repeats_and_replays_bit_for_bit(dev):
    from t2h import ops

    rows, h, d = 900, 16, 64
    (q, k, dq, dk), (gq, gk, bq, bk) = tensors(3, rows, h, d, BF16, dev)
    ws = torch.full((1 << 24,), 255, dtype=torch.uint8, device=dev)
    f = freqs(d)
    step = lambda: ops.qk_rmsnorm_rope_backward(dq=dq, dk=dk, q=q, k=k, gamma_q=gq, gamma_k=gk, bias_q=bq, bias_k=bk,
                                                freqs=f, grid_res=16, workspace=ws)
    want = step()
    for a, b in zip(step(), want):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        dq.mul_(0.5)
        q.add_(0.25)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_no_rows(dev):
    from t2h import ops

    z = torch.empty((0, 2, 64), dtype=F16, device=dev)
    gq = torch.ones((2, 64), device=dev)
    r = ops.qk_rmsnorm_rope_backward(dq=z, q=z, gamma_q=gq, bias_q=gq, use_rope=False)
    assert r[0].shape == z.shape and (r[2] == 0).all() and (r[4] == 0).all()


@pytest.mark.parametrize("dtype,h,d", [(F16, 12, 128), (BF16, 16, 64), (F32, 5, 128)])
def test_tensors_beyond_the_cache_against_pieces(dev, dtype, h, d):
    """Large tensors are read by another policy: dx is the pieces' bit for bit.
    A term g * xh of dgamma carries at most d + 8 roundings (the squares' sum, its
    root, three products), a sum less than 200 additions one behind the other in
    either form: 2 * (d + 208) 2^-24 of the terms' magnitudes."""
    from t2h import ops

    rows = (450 << 20) // (6 * h * d * torch.finfo(dtype).bits // 8)
    g = torch.Generator(device=dev).manual_seed(4)
    q, k, dq, dk = (torch.randn((rows, h, d), generator=g, device=dev).to(dtype) for _ in range(4))
    gm = torch.randn((h, d), generator=g, device=dev) * 0.1 + 1
    kw = dict(gamma_q=gm, gamma_k=gm, use_rope=False)
    got = ops.qk_rmsnorm_rope_backward(dq=dq, dk=dk, q=q, k=k, **kw)
    sums = [0.0, 0.0]
    for at in range(0, rows, 7000):
        s = slice(at, at + 7000)
        want = ops.qk_rmsnorm_rope_backward(dq=dq[s], dk=dk[s], q=q[s], k=k[s], **kw)
        assert torch.equal(got[0][s], want[0]) and torch.equal(got[1][s], want[1])
        sums = [a + b.double() for a, b in zip(sums, want[2:4])]
    for x, dy, total, want in ((q, dq, got[2], sums[0]), (k, dk, got[3], sums[1])):
        terms = (dy.double() * torch.nn.functional.normalize(x.double(), dim=-1)).abs().sum(0) * d ** 0.5
        assert ((total.double() - want).abs() <= 2 * (d + 208) * 2.0 ** -24 * terms).all()
