"""The attention branch as a training step runs it: projection, epilogue,
attention, and back through all of them into one packed gradient; the same
captured; the dense and sparse entry points; refusals that need device tensors."""
import math

import pytest
import torch

import _attention as ref
import test_gpu_qk_backward as qk

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


class Branch:
    """A self attention over a ragged batch of voxels."""

    def __init__(self, dtype, dev, lens=(70, 1, 130), heads=4, d=64, width=256):
        from t2h import nn

        g = torch.Generator().manual_seed(5)
        r = lambda *s, std=1.0: torch.randn(s, generator=g) * std
        t = sum(lens)
        self.h, self.d, self.nb = heads, d, len(lens)
        self.x = r(t, width).to(dtype).to(dev)
        self.w = r(3 * heads * d, width, std=width ** -0.5).to(dtype).to(dev)
        self.bias = [r(heads, d, std=0.1).to(dev) for _ in range(2)]
        self.gamma = [(1 + r(heads, d, std=0.1)).to(dev) for _ in range(2)]
        self.g = r(t, heads, d, std=0.1).to(dtype).to(dev)
        self.freqs = nn.rope_freqs(d)
        co = torch.randint(0, 64, (t, 4), generator=g, dtype=torch.int32)
        self.coords = co.to(dev)
        cuts = [0]
        for n in lens:
            cuts.append(cuts[-1] + n)
        self.cuts = cuts
        off = torch.tensor(cuts, device=dev)
        self.seg = dict(nbatch=self.nb, q_offsets=off, k_offsets=off)

    def step(self):
        from t2h import ops

        t, h, d = self.x.shape[0], self.h, self.d
        qkv = ops.linear(self.x, self.w).view(t, 3, h, d)
        q0, k0, v = qkv.unbind(1)
        q, k = ops.qk_rmsnorm_rope(q=q0, k=k0, gamma_q=self.gamma[0], gamma_k=self.gamma[1], bias_q=self.bias[0],
                                   bias_k=self.bias[1], freqs=self.freqs, coords=self.coords)
        out, lse = ops.attention(q, k, v, need_lse=True, **self.seg)
        dqkv = torch.empty_like(qkv)
        dq, dk, dv = dqkv.unbind(1)
        ops.attention_backward(self.g, q, k, v, out, lse, dq=dq, dk=dk, dv=dv, **self.seg)
        grads = (dq.clone(), dk.clone(), dv.clone())
        par = ops.qk_rmsnorm_rope_backward(dq=dq, dk=dk, q=q0, k=k0, gamma_q=self.gamma[0], gamma_k=self.gamma[1],
                                           bias_q=self.bias[0], bias_k=self.bias[1], freqs=self.freqs,
                                           coords=self.coords, in_place=True)
        return qkv, q, k, out, lse, *grads, dqkv, *par[2:]


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_each_stage_from_the_stored_values_before_it(dev, dtype):
    """Every stage against its definition in 64 bits on what the stage before
    stored, with that stage's own bound."""
    b = Branch(dtype, dev)
    qkv, q, k, out, lse, dq, dk, dv, dqkv, dgq, dgk, dbq, dbk = b.step()
    v, scale = qkv[:, 2], b.d ** -0.5
    seg = dict(nbatch=b.nb, q_offsets=b.cuts, k_offsets=b.cuts)
    wo, wl, bo, bl = ref.forward(q, k, v, scale, **seg)
    ref.check(out, wo, bo, "out")
    ref.check(lse, wl, bl, "lse")
    for got, (want, bound), name in zip((dq, dk, dv), ref.backward(b.g, q, k, v, out, lse, scale, **seg),
                                        ("dq", "dk", "dv")):
        ref.check(got, want, bound, name)
    assert torch.equal(dqkv[:, 2], dv)
    cs = qk.cos_sin(qkv.shape[0], b.d, b.freqs, b.coords.cpu().numpy()[:, 1:])
    for i, (dy, dg, db) in enumerate(((dq, dgq, dbq), (dk, dgk, dbk))):
        dx, edx, wg, eg, wb, eb = qk.reference(qkv[:, i], dy, b.gamma[i], b.bias[i], cs, dtype)
        qk.check(dqkv[:, i], dx, edx, "dx")
        qk.check(dg, wg, eg, "dgamma")
        qk.check(db, wb, eb, "dbias")


def test_the_whole_step_captured(dev):
    """In a graph, with the weights and inputs changed between the replays and
    eager steps in between; two branches of one shape in two graphs."""
    bs = [Branch(F16, dev), Branch(F16, dev, lens=(1, 200))]
    for b in bs:
        b.step()
    torch.cuda.synchronize()
    graphs, got = [], []
    for b in bs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(b.step())
        graphs.append(g)
    for i in range(3):
        for b in bs:
            b.x.mul_(0.9)
            b.gamma[0].add_(0.05)
            b.g.mul_(1.5)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for b, r in zip(bs, got):
            for x, y in zip(r, b.step()):
                assert torch.equal(x, y)
    torch.cuda.synchronize()


def test_overlapping_calls_on_two_streams(dev):
    """Two streams, each with its own problem and workspaces."""
    bs = [Branch(BF16, dev), Branch(BF16, dev, lens=(301,))]
    want = [b.step() for b in bs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i, (b, s) in enumerate(zip(bs, streams)):
            with torch.cuda.stream(s):
                got[i] = b.step()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_dense_entry_point(dev):
    from t2h import nn

    n, l, lk, h, d = 3, 50, 70, 2, 64
    g = torch.Generator().manual_seed(0)
    q = torch.randn((n, l, h, d), generator=g).half().to(dev)
    k, v = (torch.randn((n, lk, h, d), generator=g).half().to(dev) for _ in range(2))
    lens = torch.tensor([70, 0, 33], device=dev)
    for kl in (None, lens):
        out = nn.scaled_dot_product_attention(q, k, v, k_lens=kl)
        want, _, bound, _ = ref.forward(q.view(-1, h, d), k.view(-1, h, d), v.view(-1, h, d), d ** -0.5, nbatch=n,
                                        k_lens=None if kl is None else kl.tolist())
        ref.check(out.view(-1, h, d), want, bound, "out")
    with pytest.raises(ValueError):
        nn.scaled_dot_product_attention(q[0], k, v)
    with pytest.raises(ValueError):
        nn.scaled_dot_product_attention(q, k[:2], v[:2])


def test_sparse_entry_point(dev):
    from t2h import sparse

    g = torch.Generator().manual_seed(1)
    lens, h, d = [40, 3, 90], 2, 64
    t = sum(lens)
    co = torch.zeros((t, 4), dtype=torch.int32)
    co[:, 0] = torch.repeat_interleave(torch.arange(3), torch.tensor(lens))
    r = lambda *s: torch.randn(s, generator=g).bfloat16().to(dev)
    q = sparse.SparseTensor(r(t, h, d), co.to(dev), 3)
    k, v = q.replace(r(t, h, d)), q.replace(r(t, h, d))
    cuts = [0, 40, 43, 133]
    want, _, bound, _ = ref.forward(q.feats, k.feats, v.feats, d ** -0.5, nbatch=3, q_offsets=cuts, k_offsets=cuts)
    ref.check(sparse.sparse_scaled_dot_product_attention(q, k, v).feats, want, bound, "sparse")
    vl = [sparse.VarLenTensor(x.feats, cuts) for x in (q, k, v)]
    ref.check(sparse.sparse_scaled_dot_product_attention(*vl).feats, want, bound, "varlen")
    ctx, val = r(3, 21, h, d), r(3, 21, h, d)
    out = sparse.sparse_scaled_dot_product_attention(q, ctx, val)
    want, _, bound, _ = ref.forward(q.feats, ctx.view(-1, h, d), val.view(-1, h, d), d ** -0.5, nbatch=3, q_offsets=cuts)
    ref.check(out.feats, want, bound, "cross")
    with pytest.raises(ValueError):
        sparse.sparse_scaled_dot_product_attention(q, ctx[:2], val[:2])


def test_refusals_of_device_tensors(dev):
    from t2h import _lib, ops

    q = torch.zeros((8, 2, 64), dtype=F16, device=dev)
    out, lse = ops.attention(q, q.clone(), q.clone(), need_lse=True)
    good = dict(dout=q, q=q, k=q, v=q, out=out, lse=lse)
    off = torch.tensor([0, 8], device=dev)
    bad = [lambda: ops.attention(q, q[:, :1].expand(8, 2, 64)[:, :, :32], q),
           lambda: ops.attention(q, q, q[:4]),
           lambda: ops.attention(q, q, q.bfloat16()),
           lambda: ops.attention(q.view(8, 128), q, q),
           lambda: ops.attention(q, q, torch.zeros((8, 64, 2), dtype=F16, device=dev).transpose(1, 2)),
           lambda: ops.attention(q, q, q, nbatch=3),
           lambda: ops.attention(q, q, q, q_offsets=off.int()),
           lambda: ops.attention(q, q, q, q_offsets=off, nbatch=2),
           lambda: ops.attention(q, q, q, k_lens=off),
           lambda: ops.attention(q, q, q, scale=-1.0),
           lambda: ops.attention(q, q, q, out=q[:, :, :32]),
           lambda: ops.attention(q, q, q, out=q),
           lambda: ops.attention(q, q, q, workspace=torch.empty(64, device=dev)),
           lambda: ops.attention(q, q, torch.empty(8 * 128 + 1, dtype=F16, device=dev)[1:].view(8, 2, 64)),
           lambda: ops.attention_backward(**{**good, "lse": lse.t()}),
           lambda: ops.attention_backward(**{**good, "lse": lse.half()}),
           lambda: ops.attention_backward(**{**good, "dout": q[:4]}),
           lambda: ops.attention_backward(**good, dq=q),
           lambda: ops.attention_backward(**good, workspace=torch.empty(16, dtype=torch.uint8, device=dev)),
           lambda: ops.qk_rmsnorm_rope_backward(dq=q, gamma_q=torch.ones((2, 64), device=dev), use_rope=False),
           lambda: ops.qk_rmsnorm_rope_backward(dq=q, q=q.float(), gamma_q=torch.ones((2, 64), device=dev), use_rope=False),
           lambda: ops.qk_rmsnorm_rope_backward(dq=q, q=q, gamma_q=torch.ones((2, 32), device=dev), use_rope=False),
           lambda: ops.qk_rmsnorm_rope_backward(dq=q, dk=q[:4], use_rope=False),
           lambda: ops.qk_rmsnorm_rope_backward(dq=q, q=q, gamma_q=torch.ones((2, 64), device=dev))]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    for f in (lambda: ops.attention(q.float(), q.float(), q.float()),
              lambda: ops.attention(*(q.repeat(1, 1, 2)[:, :, :96].contiguous() for _ in range(3)))):
        with pytest.raises(_lib.T2HError):
            f()


def test_a_step_against_the_gradient_of_the_whole_branch(dev):
    """dgamma, dbias and the packed gradient of one bf16 step against autograd of
    the branch in 64 bits, from the same stored projection. Rounding q and k
    turns a score by at most 2 u |q| |k| scale, e = 2 u sqrt(D) max(gamma)^2 (u =
    2^-8; Cauchy), and a probability by a factor within exp(+-2 e); P, dS, out
    and the stored gradients add 4 u. Held against the same sums over
    magnitudes, through which the epilogue passes an error on at most twice
    (dx is a projection of w)."""
    dtype = BF16
    b = Branch(dtype, dev, lens=(60, 41))
    qkv, *_, dqkv, dgq, dgk, dbq, dbk = b.step()
    u, h, d = 2.0 ** -8, b.h, b.d
    x = qkv.cpu().double().requires_grad_()
    gm = [t.cpu().double().requires_grad_() for t in b.gamma]
    bs = [t.cpu().double().requires_grad_() for t in b.bias]
    c, s = (t[:, None] for t in qk.cos_sin(x.shape[0], d, b.freqs, b.coords.cpu().numpy()[:, 1:]))

    def epilogue(i):
        y = x[:, i] + bs[i]
        y = y / y.norm(dim=-1, keepdim=True) * gm[i] * math.sqrt(d)
        re, im = y[..., 0::2], y[..., 1::2]
        return torch.stack([re * c - im * s, re * s + im * c], -1).reshape(y.shape)

    q, k, v = epilogue(0), epilogue(1), x[:, 2]
    out = torch.zeros_like(q)
    for lo, hi in zip(b.cuts, b.cuts[1:]):
        for i in range(h):
            p = torch.softmax(q[lo:hi, i] @ k[lo:hi, i].t() * d ** -0.5, 1)
            out[lo:hi, i] = p @ v[lo:hi, i]
    (out * b.g.cpu().double()).sum().backward()
    e = 2 * u * math.sqrt(d) * max(float(t.detach().abs().max()) for t in gm) ** 2
    rel = math.expm1(2 * e) + 4 * u
    # |dS| terms: P (|dout||v| + |dout||out|), summed against |k|, |q| rows of length sqrt(D) gamma
    go = b.g.cpu().double()
    top = max(float(t.detach().abs().max()) for t in gm) * math.sqrt(d)
    vmax = float(v.detach().norm(dim=-1).max())
    gmax = float(go.norm(dim=-1).max())
    for got, want in ((dqkv, x.grad), (dgq, gm[0].grad), (dgk, gm[1].grad), (dbq, bs[0].grad), (dbk, bs[1].grad)):
        got = got.cpu().double()
        assert torch.isfinite(got).all()
        # the largest any entry's terms can sum to: a row's |dS| is at most 2 gmax vmax
        terms = 2 * gmax * vmax * d ** -0.5 * top
        lim = rel * (terms * 2 + float(want.abs().max()))
        if want.dim() == 2:
            lim *= math.sqrt(x.shape[0]) * 4        # sums over the rows, errors of either sign
        assert float((got - want).abs().max()) <= lim
        cos = float((got * want).sum() / (got.norm() * want.norm()))
        assert cos > 1 - rel ** 2 * 4
