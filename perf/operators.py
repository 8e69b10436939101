"""The attention operators and the gradients of the attention branch, as measurable cases.

A case is one pass of one operator through the public Python interface (`t2h.ops`):

- attention: softmax(scale * q k^T) v within the segments of a ragged or dense batch, with the
  log-sum-exp of each row where a training step needs it;
- attention_backward: dq, dk, dv from dout, the forward's operands, its output and its log-sum-exp,
  with the probabilities computed again;
- qk_rmsnorm_rope_backward: the gradients of the q/k epilogue (bias, per-head RMS norm, rotation) of
  the same branch, with those of gamma and bias.

Token counts are those of the sparse-structure grid (16^3 = 4,096 tokens), the structured latent
(2,369), the ragged 64^3 pair (39,804), the 128^3 shell (201,436) and an image's 1,029 condition tokens.
Heads are those of the two widths, 1536 (12 of 128) and 1024 (16 of 64).

With `own` false a pass computes the operators from elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
HEADS = {1536: (12, 128), 1024: (16, 64)}
IMAGE = 1029            # condition tokens of one image
PAIR = 39_804           # tokens of the ragged 64^3 pair
FULL = 201_436          # tokens of the 128^3 shell
MOST = 2 * 19_902 ** 2  # query-key pairs of the largest attention case


# Attention cases: q rows in `batch` segments (lengths drawn within a factor of `spread` of each
# other; 1: equal), `ctx` keys for each segment (0: self attention, keys = queries), `pad`: of a
# segment's keys only some count (k_lens), `kv` key/value heads, `layout` of the operands.
def listed():
    return [
        # one token (a pooled or register token) over an image's condition tokens: latency
        dict(name="attn_1x1029", op="attention", rows=1, batch=1, spread=1, ctx=IMAGE, pad=False, width=1024, kv=16,
             layout="rows", dtype="f16", lse=False),
        # cross attention of the structured latent, two samples, condition tokens padded to one length
        dict(name="attn_cross_2369", op="attention", rows=2369, batch=2, spread=2, ctx=IMAGE, pad=True, width=1024,
             kv=16, layout="rows", dtype="f16", lse=True),
        # self attention of the dense 16^3 grid, on the head-major operands of the attention pack
        dict(name="attn_dense_4096", op="attention", rows=4096, batch=1, spread=1, ctx=0, pad=False, width=1536, kv=12,
             layout="heads", dtype="bf16", lse=False),
        # self attention of the ragged pair in training: the packed qkv, log-sum-exp kept
        dict(name="attn_ragged_39804", op="attention", rows=PAIR, batch=2, spread=1.2, ctx=0, pad=False, width=1536,
             kv=12, layout="rows", dtype="f16", lse=True),
        # gradients within small windows of the structured latent: many short segments
        dict(name="bwd_windows_2369", op="attention_backward", rows=2369, batch=64, spread=4, ctx=0, pad=False,
             width=1024, kv=16, layout="rows", dtype="bf16"),
        # ... of the dense grid's self attention
        dict(name="bwd_dense_4096", op="attention_backward", rows=4096, batch=1, spread=1, ctx=0, pad=False,
             width=1536, kv=12, layout="rows", dtype="bf16"),
        # ... of the pair's cross attention: few keys gather from many queries
        dict(name="bwd_cross_39804", op="attention_backward", rows=PAIR, batch=2, spread=1.2, ctx=IMAGE, pad=True,
             width=1536, kv=12, layout="rows", dtype="f16"),
        # ... of the ragged pair's self attention: the most work of any case
        dict(name="bwd_ragged_39804", op="attention_backward", rows=PAIR, batch=2, spread=1.2, ctx=0, pad=False,
             width=1536, kv=12, layout="rows", dtype="f16"),
        # epilogue gradients of a handful of tokens: all latency
        dict(name="qkbwd_37", op="qk_backward", rows=37, width=1024, dtype="bf16", bias=True, pos="coords", which="q"),
        # ... of the dense grid in f32, as the reference runs it
        dict(name="qkbwd_dense_4096", op="qk_backward", rows=4096, width=1536, dtype="f32", bias=False, pos="grid",
             which="qk"),
        # ... of the whole shell's packed qkv
        dict(name="qkbwd_201k", op="qk_backward", rows=FULL, width=1536, dtype="f16", bias=True, pos="coords",
             which="qk"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention_backward", "attention_backward", "qk_backward"])
    width = rng.choice([1536, 1024])
    h, _ = HEADS[width]
    if op == "qk_backward":
        return dict(op=op, rows=_log_int(rng, 16, 150_000), width=width, dtype=rng.choice(["f32", "f16", "bf16"]),
                    bias=rng.random() < 0.5, pos=rng.choice(["coords", "grid", "none"]),
                    which=rng.choice(["q", "k", "qk"]))
    while True:
        few = rng.random() < 0.25
        rows = rng.randint(1, 64) if few else _log_int(rng, 64, PAIR)
        batch = 1 if rows < 8 else _log_int(rng, 1, max(1, min(64, rows // 8)))
        ctx = _log_int(rng, 1, 60_000 if few else 4096) if few or rng.random() < 0.5 else 0
        case = dict(op=op, rows=rows, batch=batch, spread=rng.choice([1, 2, 4]), ctx=ctx,
                    pad=ctx > 0 and rng.random() < 0.4, width=width, kv=rng.choice([h, h, h, h // 4, 1]),
                    layout=rng.choice(["rows", "rows", "heads"]) if batch == 1 else "rows",
                    dtype=rng.choice(["f16", "bf16"]))
        if op == "attention":
            case["lse"] = rng.random() < 0.5
        if batch * ctx <= FULL and _pairs(case) * width <= MOST * 1536:
            return case


# ---- sizes, from the case alone --------------------------------------------
def _lens(case):
    """Rows of each segment."""
    rows, b = case["rows"], case["batch"]
    rng = random.Random(rows * 131 + b)
    share = [rng.uniform(1.0, case["spread"]) for _ in range(b)]
    cuts = [round(rows * sum(share[:i]) / sum(share)) for i in range(b)] + [rows]
    return [cuts[i + 1] - cuts[i] for i in range(b)]


def _key_lens(case):
    """(keys held for each segment, keys that count)."""
    if not case["ctx"]:
        return _lens(case), _lens(case)
    b, ctx = case["batch"], case["ctx"]
    if not case["pad"]:
        return [ctx] * b, [ctx] * b
    rng = random.Random(ctx * 17 + b)
    used = [rng.randint(ctx // 2, ctx) for _ in range(b)]
    if b > 2:
        used[b // 2] = 0    # a sample without a condition
    return [ctx] * b, used


def _pairs(case):
    return sum(n * m for n, m in zip(_lens(case), _key_lens(case)[1]))


def _cuts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# ---- inputs, from the seed alone -------------------------------------------
class _Make:
    def __init__(self, seed: int):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.dev = torch.device("cuda")

    def randn(self, shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=self.g, device=self.dev).mul_(std).add_(mean)

    def normed(self, rows, heads, d):
        """Rows as the per-head norm leaves them (length about sqrt(d)), some heads sharper than others."""
        x = self.randn((rows, heads, d))
        x *= math.sqrt(d) / x.norm(dim=-1, keepdim=True)
        return x * torch.exp(0.4 * self.randn((heads, 1)))

    def rows(self, n, heads, d, std=1.0):
        return self.randn((n, heads, d)) * torch.exp(0.3 * self.randn((heads, d))) * std

    def voxels(self, n, res):
        """n voxels of a res^3 grid as (0, x, y, z), in the order the sparse stage lists them."""
        idx = torch.randperm(res ** 3, generator=self.g, device=self.dev)[:n].sort().values
        out = torch.zeros((n, 4), dtype=torch.int32, device=self.dev)
        out[:, 1], out[:, 2], out[:, 3] = idx // (res * res), idx // res % res, idx % res
        return out


def _freqs(d):
    n = d // 2 // 3
    return (np.float32(1.0) / np.float32(10000.0) ** (np.arange(n, dtype=np.float32) / np.float32(n))).astype(np.float32)


def _strided(parts, dtype):
    """Tensors [rows, H_i, D] as views of one packed buffer [rows, sum H_i, D]."""
    full = torch.cat([p.to(dtype) for p in parts], dim=1)
    return list(full.split([p.shape[1] for p in parts], dim=1))


def _attention_inputs(case, seed):
    mk = _Make(seed)
    h, d = HEADS[case["width"]]
    kv, dt = case["kv"], DTYPES[case["dtype"]]
    held, used = _key_lens(case)
    q = mk.normed(case["rows"], h, d)
    k, v = mk.normed(sum(held), kv, d), mk.rows(sum(held), kv, d)
    s = {"case": case, "scale": d ** -0.5}
    if case["layout"] == "heads":       # head-major [H, rows, D], the scale already in q
        q = q * d ** -0.5
        s["scale"] = 1.0
        s["q"], s["k"], s["v"] = (t.to(dt).transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    elif case["ctx"]:
        s["q"] = q.to(dt)
        s["k"], s["v"] = _strided([k, v], dt)
    else:
        s["q"], s["k"], s["v"] = _strided([q, k, v], dt)
    s["q_cuts"], s["k_cuts"], s["k_used"] = _cuts(_lens(case)), _cuts(held), used
    dev = mk.dev
    ragged = case["batch"] > 1 and not (case["spread"] == 1 and case["rows"] % case["batch"] == 0)
    s["segments"] = dict(
        nbatch=case["batch"],
        q_offsets=torch.tensor(s["q_cuts"], dtype=torch.int64, device=dev) if ragged else None,
        k_offsets=torch.tensor(s["k_cuts"], dtype=torch.int64, device=dev) if ragged and not case["ctx"] else None,
        k_lens=torch.tensor(used, dtype=torch.int64, device=dev) if case["pad"] else None)
    if case["op"] == "attention_backward":
        s["dout"] = mk.rows(case["rows"], h, d, 0.1).to(dt)
        s["out"], s["lse"] = _forward(s, True)
    return s


def _qk_inputs(case, seed):
    mk = _Make(seed)
    h, d = HEADS[case["width"]]
    t, dt = case["rows"], DTYPES[case["dtype"]]
    s = {"case": case, "freqs": _freqs(d)}
    # q and k of the packed projection, and their gradients as the attention's backward leaves them
    x = _strided([mk.rows(t, h, d), mk.rows(t, h, d), mk.rows(t, h, d)], dt)
    g = _strided([mk.rows(t, h, d, 0.1), mk.rows(t, h, d, 0.1), mk.rows(t, h, d, 0.1)], dt)
    for i, name in enumerate("qk"):
        use = name in case["which"]
        s[name] = x[i] if use else None
        s["d" + name] = g[i] if use else None
        s["gamma_" + name] = mk.randn((h, d), 0.1, 1.0) if use else None
        s["bias_" + name] = mk.randn((h, d), 0.1) if use and case["bias"] else None
    s["rope"] = dict(use_rope=case["pos"] != "none")
    if case["pos"] == "coords":
        s["rope"]["coords"] = mk.voxels(t, 64 if t <= PAIR else 128)
    elif case["pos"] == "grid":
        s["rope"]["grid_res"] = 16
    return s


def prepare(case, seed):
    return _qk_inputs(case, seed) if case["op"] == "qk_backward" else _attention_inputs(case, seed)


# ---- one pass ----------------------------------------------------------------
def _ops():
    path = os.path.join(os.getcwd(), "trellis2-mojo_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    from t2h import ops
    return ops


def run(s):
    case = s["case"]
    if case["op"] == "attention":
        if not own:
            out, lse = _forward(s, case["lse"])
            return [out, lse] if case["lse"] else [out]
        r = _ops().attention(s["q"], s["k"], s["v"], scale=s["scale"], need_lse=case["lse"], **s["segments"])
        return list(r) if case["lse"] else [r]
    if case["op"] == "attention_backward":
        if not own:
            return _backward(s)
        return list(_ops().attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], scale=s["scale"],
                                              **s["segments"]))
    if not own:
        return _qk_backward(s)
    r = _ops().qk_rmsnorm_rope_backward(dq=s["dq"], dk=s["dk"], q=s["q"], k=s["k"], gamma_q=s["gamma_q"],
                                        gamma_k=s["gamma_k"], bias_q=s["bias_q"], bias_k=s["bias_k"],
                                        freqs=s["freqs"], **s["rope"])
    return [t for t in r if t is not None]


# ---- plain forms -------------------------------------------------------------
HELD = 1 << 29      # scores held at once


def _groups(s):
    """(segment, query heads, key/value head): as many heads at once as HELD scores allow."""
    h, kv = s["q"].shape[1], s["k"].shape[1]
    for b in range(s["case"]["batch"]):
        n, m = s["q_cuts"][b + 1] - s["q_cuts"][b], s["k_used"][b]
        if n == 0:
            continue
        q_rows = slice(s["q_cuts"][b], s["q_cuts"][b + 1])
        k_rows = slice(s["k_cuts"][b], s["k_cuts"][b] + m)
        step = max(1, min(kv, HELD // max(1, n * m * (h // kv))))
        for lo in range(0, kv, step):
            hi = min(kv, lo + step)
            yield q_rows, k_rows, slice(lo * (h // kv), hi * (h // kv)), slice(lo, hi)


def _q_heads(t, rows, heads, group):
    """[rows, H, D] -> [kv heads, group * rows, D] in 32 bits."""
    x = t[rows, heads].float().transpose(0, 1)
    return x.reshape(x.shape[0] // group, group * x.shape[1], x.shape[2])


def _k_heads(t, rows, heads):
    return t[rows, heads].float().transpose(0, 1).contiguous()


def _to_rows(x, group):
    """[kv heads, group * rows, D] -> [rows, H, D]."""
    kv, n, d = x.shape
    return x.reshape(kv * group, n // group, d).transpose(0, 1)


def _forward(s, need_lse):
    q, k, v = s["q"], s["k"], s["v"]
    g = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.full((q.shape[1], q.shape[0]), float("-inf"), device=q.device) if need_lse else None
    for qr, kr, qh, kh in _groups(s):
        if kr.stop == kr.start:
            continue
        p = torch.matmul(_q_heads(q, qr, qh, g), _k_heads(k, kr, kh).transpose(1, 2).contiguous())
        p *= s["scale"]
        top = p.amax(-1, keepdim=True)
        p = p.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        out[qr, qh] = _to_rows(torch.matmul(p, _k_heads(v, kr, kh)) / total, g).to(out.dtype)
        if need_lse:
            lse[qh, qr] = (top + total.log()).reshape(-1, qr.stop - qr.start)
        del p
    return out, lse


def _backward(s):
    q, k, v = s["q"], s["k"], s["v"]
    g = q.shape[1] // k.shape[1]
    dq = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    dk, dv = (torch.zeros(k.shape, dtype=k.dtype, device=k.device) for _ in range(2))
    delta = (s["dout"].float() * s["out"].float()).sum(-1).t()
    for qr, kr, qh, kh in _groups(s):
        if kr.stop == kr.start:
            continue
        qf, kf = _q_heads(q, qr, qh, g), _k_heads(k, kr, kh)
        dof = _q_heads(s["dout"], qr, qh, g)
        rows = lambda t: t[qh, qr].reshape(kf.shape[0], -1, 1)
        p = torch.matmul(qf, kf.transpose(1, 2).contiguous()).mul_(s["scale"]).sub_(rows(s["lse"])).exp_()
        dv[kr, kh] = torch.matmul(p.transpose(1, 2), dof).transpose(0, 1).to(dv.dtype)
        dp = torch.matmul(dof, _k_heads(v, kr, kh).transpose(1, 2).contiguous())
        p *= dp.sub_(rows(delta))
        del dp
        dq[qr, qh] = _to_rows(torch.matmul(p, kf).mul_(s["scale"]), g).to(dq.dtype)
        dk[kr, kh] = torch.matmul(p.transpose(1, 2), qf).mul_(s["scale"]).transpose(0, 1).to(dk.dtype)
        del p
    return [dq, dk, dv]


def _angles(s, rows, d):
    """Angle of each (row, slot) in f32: position times frequency, one rounding; 0 in unrotated slots."""
    dev = torch.device("cuda")
    ang = torch.zeros((rows, d // 2), device=dev)
    if not s["rope"]["use_rope"]:
        return ang
    if "coords" in s["rope"]:
        pos = s["rope"]["coords"][:, 1:4].float()
    else:
        res = s["rope"]["grid_res"]
        i = torch.arange(rows, device=dev) % res ** 3
        pos = torch.stack([i // (res * res), i // res % res, i % res], 1).float()
    f = torch.from_numpy(s["freqs"]).to(dev)
    ang[:, :3 * f.numel()] = (pos[:, :, None] * f).reshape(rows, -1)
    return ang


def _qk_backward(s):
    dxs, dgs, dbs = [], [], []
    for name in s["case"]["which"]:
        x, gy = s[name].float(), s["d" + name].float()
        rows, h, d = x.shape
        if s["bias_" + name] is not None:
            x = x + s["bias_" + name]
        if s["rope"]["use_rope"]:
            ang = _angles(s, rows, d).double()
            c, sn = ang.cos().float()[:, None], ang.sin().float()[:, None]
            re, im = gy[..., 0::2], gy[..., 1::2]
            gy = torch.stack([re * c + im * sn, im * c - re * sn], -1).reshape(rows, h, d)
        n = (x * x).sum(-1, keepdim=True).sqrt().clamp_min(1e-12)
        xh = x / n
        dgs.append((gy * xh).mul_(math.sqrt(d)).sum(0, dtype=torch.float64).float())
        w = gy * (s["gamma_" + name] * math.sqrt(d))
        dx = (w - xh * (w * xh).sum(-1, keepdim=True)) / n
        dxs.append(dx.to(s[name].dtype))
        if s["bias_" + name] is not None:
            dbs.append(dx.sum(0, dtype=torch.float64).float())
    return [*dxs, *dgs, *dbs]


# ---- what a pass cannot do without -------------------------------------------
def work(case):
    e = SIZE[case["dtype"]]
    h, d = HEADS[case["width"]]
    if case["op"] == "qk_backward":
        n, t = len(case["which"]), case["rows"]
        params = n * h * d * 4 * (2 + 2 * case["bias"])
        return {"bytes": n * 3 * e * t * h * d + params + (16 * t if case["pos"] == "coords" else 0),
                "flops": n * t * h * (d * 15 + 10)}
    rows, keys = case["rows"], sum(_key_lens(case)[1])
    q, kv = e * rows * h * d, e * keys * case["kv"] * d
    if case["op"] == "attention":
        return {"bytes": 2 * q + 2 * kv + (4 * rows * h if case["lse"] else 0), "flops": 4 * d * h * _pairs(case)}
    held = e * sum(_key_lens(case)[0]) * case["kv"] * d
    return {"bytes": 4 * q + 2 * kv + 2 * held + 4 * rows * h, "flops": 10 * d * h * _pairs(case)}


# ---- the same from the definitions, in 64 bits ---------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "qk_backward":
        return _exact_qk(s)
    q, k, v = s["q"], s["k"], s["v"]
    (t, h, d), group = q.shape, q.shape[1] // k.shape[1]
    back = case["op"] == "attention_backward"
    f64 = dict(dtype=torch.float64, device=q.device)
    out, lse = torch.zeros((t, h, d), **f64), torch.full((h, t), -math.inf, **f64)
    dk, dv = torch.zeros(k.shape, **f64), torch.zeros(v.shape, **f64)
    for b in range(case["batch"]):
        m = s["k_used"][b]
        if m == 0:
            continue
        k0, hi = s["k_cuts"][b], s["q_cuts"][b + 1]
        step = max(1, HELD // 4 // m)
        for lo in range(s["q_cuts"][b], hi, step):
            rows = slice(lo, min(hi, lo + step))
            for i in range(h):
                j = i // group
                qi, kj, vj = q[rows, i].double(), k[k0:k0 + m, j].double(), v[k0:k0 + m, j].double()
                score = qi @ kj.t().contiguous() * s["scale"]
                if not back:
                    lse[i, rows] = torch.logsumexp(score, 1)
                    out[rows, i] = torch.softmax(score, 1) @ vj
                    continue
                prob = torch.exp(score - s["lse"][i, rows].double()[:, None])
                do = s["dout"][rows, i].double()
                dv[k0:k0 + m, j] += prob.t().contiguous() @ do
                inner = (do * s["out"][rows, i].double()).sum(1, keepdim=True)
                ds = prob * (do @ vj.t().contiguous() - inner) * s["scale"]
                out[rows, i] = ds @ kj
                dk[k0:k0 + m, j] += ds.t().contiguous() @ qi
    if back:
        return [out, dk, dv]
    return [out, lse] if case["lse"] else [out]


def _exact_qk(s):
    dxs, dgs, dbs = [], [], []
    for name in s["case"]["which"]:
        rows, h, d = s[name].shape
        x = s[name].double()
        if s["bias_" + name] is not None:
            x = x + s["bias_" + name].double()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), -_angles(s, rows, d).double())
        gy = s["d" + name].double().reshape(rows, h, d // 2, 2)
        gy = torch.view_as_real(torch.view_as_complex(gy.contiguous()) * turn[:, None]).reshape(rows, h, d)
        length = torch.linalg.vector_norm(x, dim=-1, keepdim=True).clamp_min(1e-12)
        unit = x / length
        dgs.append((gy * unit).sum(0) * math.sqrt(d))
        w = gy * s["gamma_" + name].double() * math.sqrt(d)
        dx = (w - unit * (w * unit).sum(-1, keepdim=True)) / length
        dxs.append(dx)
        if s["bias_" + name] is not None:
            dbs.append(dx.sum(0))
    return [*dxs, *dgs, *dbs]
