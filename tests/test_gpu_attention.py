"""Attention and its backward pass against their definitions in 64 bits."""
import math

import pytest
import torch

import _attention as ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(seed, rows, krows, h, kvh, d, dtype, dev, sharp=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda n, heads, std=1.0: (torch.randn((n, heads, d), generator=g) * std).to(dtype).to(dev)
    return r(rows, h, sharp), r(krows, kvh), r(krows, kvh), r(rows, h, 0.5)


def offs(lens, dev):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out, torch.tensor(out, dtype=torch.int64, device=dev)


def run_both(q, k, v, g, scale, dev, **seg):
    """Forward and backward against the bounds; returns what the kernels gave."""
    from t2h import ops

    host = {n: t.cpu().tolist() if isinstance(t, torch.Tensor) else t for n, t in seg.items()}
    out, lse = ops.attention(q, k, v, scale=scale, need_lse=True, **seg)
    wo, wl, bo, bl = ref.forward(q, k, v, scale, **host)
    ref.check(out, wo, bo, "out")
    ref.check(lse, wl, bl, "lse")
    grads = ops.attention_backward(g, q, k, v, out, lse, scale=scale, **seg)
    for x, (want, bound), name in zip(grads, ref.backward(g, q, k, v, out, lse, scale, **host), ("dq", "dk", "dv")):
        ref.check(x, want, bound, name)
    return out, lse, grads


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,krows", [(1, 1), (1, 64), (1, 300), (16, 65), (33, 31), (64, 64), (65, 127), (257, 129),
                                        (300, 1)])
def test_sizes(dev, dtype, d, rows, krows):
    run_both(*make(rows + krows, rows, krows, 2, 2, d, dtype, dev), d ** -0.5, dev)


@pytest.mark.parametrize("dtype,d", [(F16, 128), (BF16, 64)])
def test_self_attention_of_a_packed_qkv(dev, dtype, d):
    """q, k, v as views of [rows, 3, H, D]; gradients into views of such a buffer."""
    from t2h import ops

    rows, h = 531, 4
    qkv = torch.randn((rows, 3, h, d), generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
    q, k, v = qkv.unbind(1)
    g = make(2, rows, rows, h, h, d, dtype, dev)[3]
    out, lse, grads = run_both(q, k, v, g, d ** -0.5, dev)
    dqkv = torch.empty_like(qkv)
    dq, dk, dv = dqkv.unbind(1)
    ops.attention_backward(g, q, k, v, out, lse, dq=dq, dk=dk, dv=dv)
    for a, b in zip((dq, dk, dv), grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_head_major_operands_of_the_pack(dev, dtype):
    """The pack's [H, rows, D] outputs, the scale already in q."""
    from t2h import ops

    rows, h, d, mp = 200, 4, 64, 256
    x = torch.randn((rows, 3, h, d), generator=torch.Generator().manual_seed(3)).to(dtype).to(dev)
    qh, kh, vh = ops.attn_pack(*x.unbind(1), mp=mp, lp=mp, use_rope=False, k_transposed=False)
    q, k, v = (t.transpose(0, 1)[:rows] for t in (qh, kh, vh))
    out = ops.attention(q, k, v, scale=1.0)
    wo, _, bo, _ = ref.forward(q, k, v, 1.0)
    ref.check(out, wo, bo, "out")
    # gradients in that layout too
    g = make(4, rows, rows, h, h, d, dtype, dev)[3]
    out, lse = ops.attention(q, k, v, scale=1.0, need_lse=True)
    dq = torch.full((h, mp, d), 7.0, dtype=dtype, device=dev)
    got = ops.attention_backward(g, q, k, v, out, lse, scale=1.0, dq=dq.transpose(0, 1)[:rows])
    for t, (want, bound), name in zip(got, ref.backward(g, q, k, v, out, lse, 1.0), ("dq", "dk", "dv")):
        ref.check(t, want, bound, name)
    assert (dq[:, rows:] == 7.0).all()


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("h,kvh", [(4, 2), (6, 1)])
def test_shared_heads(dev, dtype, d, h, kvh):
    run_both(*make(5, 130, 201, h, kvh, d, dtype, dev), d ** -0.5, dev)


@pytest.mark.parametrize("dtype,d", [(F16, 128), (BF16, 64)])
def test_ragged_segments_with_empty_ones(dev, dtype, d):
    """Segments of queries without keys, keys without queries, both; a gap
    before the first and rows behind the last, which are left as they were."""
    from t2h import ops

    ql, kl = [5, 0, 64, 33, 257, 1, 0, 17], [9, 12, 0, 65, 300, 1, 0, 64]
    qo, _ = offs(ql, dev)
    ko, _ = offs(kl, dev)
    qo, ko = [x + 3 for x in qo], [x + 2 for x in ko]
    rows, krows = qo[-1] + 11, ko[-1] + 7
    q, k, v, g = make(6, rows, krows, 2, 2, d, dtype, dev)
    seg = dict(nbatch=len(ql), q_offsets=torch.tensor(qo, device=dev), k_offsets=torch.tensor(ko, device=dev))
    run_both(q, k, v, g, d ** -0.5, dev, **seg)
    # NaN in the uncovered rows of every input changes nothing and reaches nothing
    for t, o in ((q, qo), (k, ko), (v, ko), (g, qo)):
        t[:o[0]] = math.nan
        t[o[-1]:] = math.nan
    out = torch.full_like(q, 7.0)
    ops.attention(q, k, v, out=out, **seg)
    assert (out[:qo[0]] == 7.0).all() and (out[qo[-1]:] == 7.0).all()
    out, lse = ops.attention(q, k, v, need_lse=True, **seg)
    dq, dk, dv = (torch.full_like(t, 7.0) for t in (q, k, v))
    ops.attention_backward(g, q, k, v, out, lse, dq=dq, dk=dk, dv=dv, **seg)
    host = dict(nbatch=len(ql), q_offsets=qo, k_offsets=ko)
    for t, (want, bound), o, name in zip((dq, dk, dv), ref.backward(g, q, k, v, out, lse, d ** -0.5, **host),
                                         (qo, ko, ko), ("dq", "dk", "dv")):
        ref.check(t, want, bound, name)
        assert (t[:o[0]] == 7.0).all() and (t[o[-1]:] == 7.0).all()


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (F16, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 60000.0])
def test_key_lengths_and_what_lies_behind_them(dev, dtype, d, bad):
    """A padded dense batch: keys past k_lens hold anything, get zero
    gradients, and a sample of length 0 gives zeros and lse -inf."""
    from t2h import ops

    n, lq, lk, h = 5, 40, 150, 2
    q, k, v, g = make(7, n * lq, n * lk, h, h, d, dtype, dev)
    lens = [150, 0, 1, 64, 97]
    kl = torch.tensor(lens, device=dev)
    seg = dict(nbatch=n, k_lens=kl)
    clean = run_both(q, k, v, g, d ** -0.5, dev, **seg)
    for b, m in enumerate(lens):
        k[b * lk + m:(b + 1) * lk] = bad
        v[b * lk + m:(b + 1) * lk] = bad
    out, lse = ops.attention(q, k, v, need_lse=True, **seg)
    grads = ops.attention_backward(g, q, k, v, out, lse, **seg)
    for a, b in zip((out, lse, *grads), (*clean[:2], *clean[2])):
        assert torch.equal(a, b)
    assert (out[lq:2 * lq] == 0).all() and torch.isinf(lse[:, lq:2 * lq]).all()
    # lengths past the segment and below zero
    kl2 = torch.tensor([1 << 40, -5, 1, 64, 97], device=dev)
    k.nan_to_num_(0.0, 0.0, 0.0), v.nan_to_num_(0.0, 0.0, 0.0)
    a = ops.attention(q, k, v, nbatch=n, k_lens=kl2)
    b = ops.attention(q, k, v, nbatch=n, k_lens=kl)
    assert torch.equal(a, b)


def test_offsets_outside_the_tensor_stay_inside_it(dev):
    """Offsets that pass the tensors' rows or run backwards are cut to them."""
    from t2h import ops

    q, k, v, g = make(8, 100, 90, 2, 2, 64, F16, dev)
    good = torch.tensor([0, 60, 100], device=dev)
    wild = torch.tensor([0, 60, 1 << 40], device=dev)
    kgood, kwild = torch.tensor([0, 50, 90], device=dev), torch.tensor([0, 50, 1 << 50], device=dev)
    a = ops.attention(q, k, v, nbatch=2, q_offsets=good, k_offsets=kgood)
    b = ops.attention(q, k, v, nbatch=2, q_offsets=wild, k_offsets=kwild)
    assert torch.equal(a, b)
    back = torch.tensor([70, 20, -9], device=dev)
    out, lse = ops.attention(q, k, v, nbatch=2, q_offsets=back, k_offsets=back, need_lse=True)
    ops.attention_backward(g, q, k, v, out, lse, nbatch=2, q_offsets=back, k_offsets=back)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,krows,h,kvh,d", [(1, 4100, 2, 2, 128), (3, 5000, 4, 1, 64), (40, 2049, 2, 2, 64),
                                                (3000, 40, 1, 1, 128), (2500, 65, 4, 2, 64)])
def test_split_and_unsplit(dev, dtype, rows, krows, h, kvh, d):
    """Few rows over many keys (and the reverse for dk, dv): the split forms
    against the definition, and against the unsplit one up to rounding."""
    from t2h import ops

    q, k, v, g = make(9, rows, krows, h, kvh, d, dtype, dev, sharp=2.0)
    run_both(q, k, v, g, d ** -0.5, dev)
    none = torch.empty(0, dtype=torch.uint8, device=dev)
    out, lse = ops.attention(q, k, v, need_lse=True, workspace=none)
    wo, wl, bo, bl = ref.forward(q, k, v, d ** -0.5)
    ref.check(out, wo, bo, "unsplit out")
    ref.check(lse, wl, bl, "unsplit lse")


def test_split_ragged(dev):
    """Splits over segments of very different key counts, one empty."""
    ql, kl = [2, 1, 3, 4], [3000, 0, 10, 400]
    (_, qo), (_, ko) = offs(ql, dev), offs(kl, dev)
    q, k, v, g = make(10, sum(ql), sum(kl), 2, 2, 128, BF16, dev)
    run_both(q, k, v, g, 128 ** -0.5, dev, nbatch=4, q_offsets=qo, k_offsets=ko)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scores_that_rise_and_fall(dev, dtype):
    """Running maxima: keys in rising, falling and shuffled order of score, large scores of both signs."""
    d, n = 64, 400
    q, k, v, g = make(11, 48, n, 1, 1, d, dtype, dev)
    ramp = torch.linspace(-30, 30, n, device=dev)
    for order in (ramp, ramp.flip(0), ramp[torch.randperm(n, generator=torch.Generator().manual_seed(0)).to(dev)]):
        kk = (q[0, 0].float() / q[0, 0].float().norm() * order[:, None])[:, None].to(dtype)
        run_both(q, kk, v, g, 1.0, dev)
    # every score far below zero: the first maximum is the row's own
    kk = (-40.0 * q[:1, 0].float() / q[0, 0].float().norm()).expand(n, d)[:, None].to(dtype).contiguous()
    run_both(q[:1].contiguous(), kk, v, g[:1].contiguous(), 1.0, dev)


def test_small_probabilities_keep_their_precision_in_f16(dev):
    """40,000 keys of like score: P = 2.5e-5 and dS far below it are under
    f16's smallest normal number; the gradients keep the type's precision.
    dS is held to 2^-37 of |dout| |v|, a probability to 2^-39."""
    from t2h import ops

    n, d = 40_000, 64
    g0 = torch.Generator().manual_seed(12)
    q = (torch.randn((16, 1, d), generator=g0) * 0.1).half().to(dev)
    k = torch.randn((n, 1, d), generator=g0).half().to(dev)
    v = torch.randn((n, 1, d), generator=g0).half().to(dev)
    g = torch.randn((16, 1, d), generator=g0).half().to(dev)
    run_both(q, k, v, g, d ** -0.5, dev)
    out, lse = ops.attention(q, k, v, need_lse=True)
    # dv is below f16's normal numbers itself: compare it scaled, through a larger dout
    big = (g.float() * 4096).half()
    got = ops.attention_backward(big, q, k, v, out, lse)
    for t, (want, bound), name in zip(got, ref.backward(big, q, k, v, out, lse, d ** -0.5), ("dq", "dk", "dv")):
        ref.check(t, want, bound, name)


def test_one_large_row_of_dout_does_not_cost_the_others_their_gradients(dev):
    q, k, v, g = make(13, 200, 200, 1, 1, 128, F16, dev)
    g *= 0.01
    g[7] *= 1000.0
    run_both(q, k, v, g, 128 ** -0.5, dev)


def test_nan_and_infinite_inputs_stay_in_their_segment_and_head(dev):
    from t2h import ops

    for dtype in (F16, BF16):
        q, k, v, g = make(14, 120, 120, 2, 2, 64, dtype, dev)
        seg = dict(nbatch=3)
        out, lse = ops.attention(q, k, v, need_lse=True, **seg)
        clean = ops.attention_backward(g, q, k, v, out, lse, **seg)
        for bad in (math.nan, math.inf):
            q2, k2, v2, g2 = q.clone(), k.clone(), v.clone(), g.clone()
            k2[45, 0, 3] = bad
            v2[50, 0, 5] = bad
            g2[60, 0, 1] = bad
            o2, l2 = ops.attention(q2, k2, v2, need_lse=True, **seg)
            got = ops.attention_backward(g2, q2, k2, v2, out, lse, **seg)
            for a, b in zip((o2, *got), (out, *clean)):
                assert torch.equal(a[:40], b[:40]) and torch.equal(a[80:], b[80:])
                assert torch.equal(a[40:80, 1], b[40:80, 1])
            assert not torch.isfinite(o2[40:80, 0]).all()


def test_keys_past_four_gigabytes(dev):
    """Rows 8 MB apart: byte offsets beyond 32 bits within one segment."""
    from t2h import ops

    rows, d = 700, 64
    buf = torch.zeros((rows * (1 << 22) + d,), dtype=F16, device=dev)
    k = buf.as_strided((rows, 1, d), (1 << 22, d, 1))
    q, kk, v, g = make(15, 20, rows, 1, 1, d, F16, dev)
    k.copy_(kk)
    out, lse = ops.attention(q, k, v, need_lse=True)
    got = ops.attention_backward(g, q, k, v, out, lse)
    o2, l2 = ops.attention(q, kk, v, need_lse=True)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    for a, b in zip(got, ops.attention_backward(g, q, kk, v, o2, l2)):
        assert torch.equal(a, b)


def test_repeats_bit_for_bit_and_on_another_stream(dev):
    from t2h import ops

    q, k, v, g = make(16, 700, 650, 4, 2, 128, F16, dev)
    out, lse = ops.attention(q, k, v, need_lse=True)
    want = (out, lse, *ops.attention_backward(g, q, k, v, out, lse))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ws = torch.full((ops.attention_backward_workspace(700, 650, 4, 2, 128),), 255, dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    for s in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(s):
            for _ in range(2):
                o, l = ops.attention(q, k, v, need_lse=True)
                got = (o, l, *ops.attention_backward(g, q, k, v, o, l, workspace=ws))
        s.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_captured_and_replayed(dev):
    """Forward and backward of two shapes (one split) in a graph, inputs
    rewritten between the replays."""
    from t2h import ops

    sets = [make(17, 300, 280, 2, 2, 64, BF16, dev), make(18, 2, 3000, 2, 1, 128, F16, dev)]
    ws = [(torch.empty(ops.attention_workspace(q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2]),
                       dtype=torch.uint8, device=dev),
           torch.empty(ops.attention_backward_workspace(q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2]),
                       dtype=torch.uint8, device=dev)) for q, k, v, g in sets]

    def step():
        res = []
        for (q, k, v, g), (w1, w2) in zip(sets, ws):
            out, lse = ops.attention(q, k, v, need_lse=True, workspace=w1)
            res += [out, lse, *ops.attention_backward(g, q, k, v, out, lse, workspace=w2)]
        return res

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        for t in (t for s in sets for t in s):
            t.mul_(0.9).add_(0.01 * i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_no_keys_and_no_rows(dev):
    from t2h import ops

    q, k, v, g = make(19, 20, 0, 2, 2, 64, F16, dev)
    out, lse = ops.attention(q, k, v, need_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = ops.attention_backward(g, q, k, v, out, lse)
    assert (dq == 0).all() and dk.shape[0] == 0
    q, k, v, g = make(20, 0, 20, 2, 2, 64, BF16, dev)
    out, lse = ops.attention(q, k, v, need_lse=True)
    dq, dk, dv = ops.attention_backward(g, q, k, v, out, lse)
    assert out.shape[0] == 0 and (dk == 0).all() and (dv == 0).all()


def test_gradients_against_differences(dev):
    """d(sum(out * g)) along random directions: the kernels' gradients against
    central differences of the definition in 64 bits. The gradients' own error
    bound, summed over the direction, plus the difference's h^2 term."""
    d, h = 64, 2
    q, k, v, g = make(21, 50, 70, h, 1, d, BF16, dev)
    out, lse, grads = run_both(q, k, v, g, d ** -0.5, dev)
    wants = ref.backward(g, q, k, v, out, lse, d ** -0.5)
    # out's rounding enters delta: |d delta| <= sum |dout| u |out|
    u = ref.U[BF16]
    gen = torch.Generator().manual_seed(0)
    x = [t.cpu().double() for t in (q, k, v)]
    for i in range(3):
        dirn = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
        step = 1e-4

        def value(sign):
            y = list(x)
            y[i] = y[i] + sign * step * dirn
            o = torch.empty_like(x[0])
            for hh in range(h):
                p = torch.softmax(y[0][:, hh] @ y[1][:, 0].t() * d ** -0.5, 1)
                o[:, hh] = p @ y[2][:, 0]
            return (o * g.cpu().double()).sum()

        want = (value(1) - value(-1)) / (2 * step)
        got = (grads[i].cpu().double() * dirn).sum()
        slack = (wants[i][1] * dirn.abs()).sum()
        if i < 2:
            go, oo = g.cpu().double().abs(), out.cpu().double().abs()
            wobble = u * (go * oo).sum(-1)                      # [rows, H]
            for hh in range(h):
                p = torch.softmax(x[0][:, hh] @ x[1][:, 0].t() * d ** -0.5, 1)
                e = p * wobble[:, hh:hh + 1] * d ** -0.5
                slack += (e @ x[1][:, 0].abs() * dirn[:, hh].abs()).sum() if i == 0 else \
                    (e.t() @ x[0][:, hh].abs() * dirn[:, 0].abs()).sum()
        assert abs(got - want) <= slack + 1e-5 * abs(want) + 1e-6, (i, float(got), float(want), float(slack))


def test_offsets_far_below_zero_stay_inside(dev):
    """Negative offsets count as 0, in the row bounds of f16 too."""
    from t2h import ops

    q, k, v, g = make(22, 50, 40, 2, 2, 64, F16, dev)
    neg = torch.tensor([-(1 << 50), 50], device=dev)
    kneg = torch.tensor([-(1 << 45), 40], device=dev)
    out, lse = ops.attention(q, k, v, q_offsets=neg, k_offsets=kneg, need_lse=True)
    got = (out, lse, *ops.attention_backward(g, q, k, v, out, lse, q_offsets=neg, k_offsets=kneg))
    o2, l2 = ops.attention(q, k, v, need_lse=True)
    for a, b in zip(got, (o2, l2, *ops.attention_backward(g, q, k, v, o2, l2))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 16, 40])
def test_nan_keys_that_fill_a_part_of_a_tile(dev, rows, d):
    """Keys are dealt out to waves: a wave whose scores are all NaN is no wave without keys."""
    from t2h import ops

    for bad in (slice(32, 64), slice(0, 32), slice(40, 41), slice(96, 130), slice(0, 1024)):
        for krows in (130, 1024):
            q, k, v, _ = make(9, rows, krows, 2, 2, d, F16, dev)
            k[bad] = math.nan
            out, lse = ops.attention(q, k, v, need_lse=True)
            assert out.isnan().all() and lse.isnan().all(), (bad, krows)
    q, k, v, _ = make(9, rows, 5000, 2, 2, d, F16, dev)      # and in a split's part
    k[2048:2112] = math.nan
    out, lse = ops.attention(q, k, v, need_lse=True)
    assert out.isnan().all() and lse.isnan().all()


@pytest.mark.parametrize("rows,d", [(1, 64), (5, 128), (64, 64)])
def test_rows_far_apart(dev, rows, d):
    """The largest row stride: a tile's last row is 2^31 bytes from its first."""
    from t2h import ops

    stride, n = 1 << 22, 300
    q, k, v, g = make(3, rows, n, 1, 1, d, BF16, dev)
    big = torch.empty(((n - 1) * stride + 2 * d,), dtype=BF16, device=dev)
    kk, vv = (big.as_strided((n, 1, d), (stride, d, 1), at).copy_(t) for at, t in ((0, k), (d, v)))
    out, lse, _ = run_both(q, kk, vv, g, d ** -0.5, dev)
    again, _ = ops.attention(q, k, v, scale=d ** -0.5, need_lse=True)
    assert torch.equal(out, again)


def test_expanded_gradients_and_aliases_are_refused(dev):
    from t2h import ops

    q, k, v, g = make(3, 20, 20, 2, 2, 64, F16, dev)
    out, lse = ops.attention(q, k, v, need_lse=True)
    for bad in (g[:1].expand(20, 2, 64), g[:, :1].expand(20, 2, 64)):
        with pytest.raises(ValueError, match="must not be expanded"):
            ops.attention_backward(bad, q, k, v, out, lse)
        with pytest.raises(ValueError, match="must not be expanded"):
            ops.attention(bad, k, v)
    with pytest.raises(ValueError, match="unit stride"):
        ops.attention_backward(g[:, :, :1].expand(20, 2, 64), q, k, v, out, lse)
    with pytest.raises(ValueError, match="rows must not overlap"):
        ops.qk_rmsnorm_rope_backward(dq=g[:1].expand(20, 2, 64), use_rope=False)
    dq = torch.empty_like(q)
    with pytest.raises(Exception, match="alias each other"):
        ops.attention_backward(g, q, k, v, out, lse, dq=dq, dk=dq)
    with pytest.raises(Exception, match="must not alias"):
        ops.qk_rmsnorm_rope_backward(dq=g, dk=g, use_rope=False, in_place=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,krows", [(0, 1000), (1000, 0), (0, 20)])
def test_segments_of_a_tensor_without_rows(dev, dtype, rows, krows):
    """Offsets over an empty side, the other long enough to be split."""
    from t2h import ops

    q, k, v, g = make(21, rows, krows, 2, 2, 64, dtype, dev)
    seg = dict(nbatch=2, q_offsets=offs([rows // 2] * 2, dev)[1], k_offsets=offs([krows // 2] * 2, dev)[1])
    out, lse = ops.attention(q, k, v, need_lse=True, **seg)
    assert (out == 0).all() and (lse == -math.inf).all()
    for x in ops.attention_backward(g, q, k, v, out, lse, **seg):
        assert (x == 0).all()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,rows,krows,h,kvh,d", [
    (F16, 512, 512, 4, 4, 64), (BF16, 512, 512, 4, 2, 128),      # both sides in parts
    (F16, 64, 1029, 2, 2, 64), (BF16, 1029, 64, 2, 2, 128),      # one side in parts, either side's blocks first
    (F16, 2000, 512, 2, 1, 128), (BF16, 300, 3000, 12, 12, 128), (F16, 3000, 300, 12, 4, 64)])
def test_backward_forms_and_parts(dev, dtype, rows, krows, h, kvh, d):
    q, k, v, g = make(31, rows, krows, h, kvh, d, dtype, dev)
    run_both(q, k, v, g, d ** -0.5, dev)
    third = rows // 3
    _, qo = offs([third, 0, rows - third - 7], dev)              # and ragged, with uncovered rows
    _, ko = offs([krows - 9, 4, 5], dev)
    run_both(q, k, v, g, d ** -0.5, dev, nbatch=3, q_offsets=qo, k_offsets=ko)
