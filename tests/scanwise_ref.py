"""Plain 64-bit forms of the scan-wise operators, their gradients by formula, and how far a 32-bit (or 16-bit) computation of them may be
off: every bound below counts roundings of half a step (u = 2^-24 for fp32, eps(T) / 2 for the operands' type) through the formulas."""
import math

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def ranges(lengths, gaps=None):
    """[S, 2] row ranges with `gaps[i]` rows of no scan in front of scan i."""
    out, at = [], 0
    for i, n in enumerate(lengths):
        at += 0 if gaps is None else gaps[i]
        out.append((at, at + n))
        at += n
    return torch.tensor(out, dtype=torch.int32).reshape(-1, 2)


def group_norm_ref(x, groups, weight, bias, seg, eps, act, dy=None):
    """(values, bounds), each a dict of y and -- with dy -- dx, dw, db."""
    uT = half_step(x.dtype)
    xd = x.double()
    m, c = x.shape
    w = torch.ones(c, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    val = {"y": torch.zeros_like(xd), "dx": torch.zeros_like(xd), "dw": torch.zeros_like(w), "db": torch.zeros_like(w)}
    bnd = {k: torch.zeros_like(v) for k, v in val.items()}
    for lo, hi in ([(0, m)] if seg is None else seg.tolist()):
        if hi <= lo:
            continue
        n = (hi - lo) * (c // groups)
        xs = xd[lo:hi]
        g = xs.reshape(hi - lo, groups, -1)
        wide = lambda t: t.repeat_interleave(c // groups)
        mean, var = wide(g.mean((0, 2))), wide(g.var((0, 2), unbiased=False))
        rstd = (var + eps).rsqrt()
        xh = (xs - mean) * rstd
        z = xh * w + b
        # x - mean (the mean rounded once), times rstd w (three roundings), plus b: each a half step of its result
        dz_b = U32 * (6 * (xh * w).abs() + z.abs() + 2 * (mean * rstd * w).abs() + b.abs())
        sig = torch.sigmoid(z)
        slope = {None: torch.ones_like(z), "relu": (z > 0).double(), "silu": sig * (1 + z * (1 - sig))}[act]
        y = {None: z, "relu": z.clamp(min=0), "silu": z * sig}[act]
        # silu: slope at most 1.1; exp2 (1 ulp, its argument z log2 e off by |z| u), reciprocal (1 ulp), sum and product: (8 + 2 |z|) u
        act_b = dz_b if act != "silu" else 1.1 * dz_b + y.abs() * U32 * (8 + 2 * z.abs())
        val["y"][lo:hi], bnd["y"][lo:hi] = y, act_b + uT * (y.abs() + act_b)
        if dy is None:
            continue
        d = dy[lo:hi].double() * slope
        # the slope: second derivative at most 0.5 (silu), its own roundings at most 16 u (1 + |z|)
        d_b = dy[lo:hi].double().abs() * ((0.5 * dz_b + 16 * U32 * (1 + z.abs())) if act == "silu" else 0) + U32 * d.abs()
        xh_b = U32 * (3 * xh.abs() + (mean * rstd).abs())
        val["db"] += d.sum(0)
        val["dw"] += (d * xh).sum(0)
        bnd["db"] += d_b.sum(0)
        bnd["dw"] += (d_b * xh.abs() + d.abs() * xh_b).sum(0)
        t, t_b = d * w, d_b * w.abs() + U32 * (d * w).abs()
        fold = lambda u: wide(u.reshape(hi - lo, groups, -1).sum((0, 2)) / n)
        ma, mb = fold(t), fold(t * xh)
        ma_b, mb_b = fold(t_b) + U32 * ma.abs(), fold(t_b * xh.abs() + t.abs() * xh_b) + U32 * mb.abs()
        dx = rstd * (t - ma - xh * mb)
        dx_b = rstd * (t_b + ma_b + xh.abs() * mb_b + xh_b * mb.abs() + 6 * U32 * (t.abs() + ma.abs() + (xh * mb).abs()))
        val["dx"][lo:hi], bnd["dx"][lo:hi] = dx, dx_b + uT * (dx.abs() + dx_b)
    bnd["db"] += U32 * val["db"].abs()
    bnd["dw"] += U32 * val["dw"].abs()
    return val, bnd


def distance2(cq, ck):
    return (cq[:, None, 1:].long() - ck[None, :, 1:].long()).square().sum(-1)


def attention_ref(q, k, v, seg_q=None, seg_k=None, cq=None, ck=None, slopes=None, bias=None, edges=None, scale=None, go=None):
    """(values, bounds) of out and -- with go -- dq, dk, dv, dt."""
    uT = half_step(q.dtype)
    uP = 0.0 if q.dtype == torch.float32 else uT          # probabilities / score gradients rounded to the operands' type
    (mq, heads, dim), (mk, kv_heads, _) = q.shape, k.shape
    share = heads // kv_heads
    scale = 1 / math.sqrt(dim) if scale is None else scale
    f64 = dict(dtype=torch.float64, device=q.device)
    val = {"out": torch.zeros(q.shape, **f64), "dq": torch.zeros(q.shape, **f64), "dk": torch.zeros(k.shape, **f64), "dv": torch.zeros(k.shape, **f64),
           "dt": torch.zeros((1 if bias is None else bias.shape[0], heads), **f64)}
    bnd = {n: torch.zeros_like(t) for n, t in val.items()}
    for (q0, q1), (k0, k1) in zip([(0, mq)] if seg_q is None else seg_q.tolist(), [(0, mk)] if seg_k is None else seg_k.tolist()):
        if q1 <= q0 or k1 <= k0:
            continue
        d2 = which = None
        if slopes is not None or bias is not None:
            d2 = distance2(cq[q0:q1], ck[k0:k1])
        if bias is not None:
            which = torch.bucketize(d2, torch.tensor(edges, dtype=torch.int64, device=q.device), right=True)
        for h in range(heads):
            Q, K, V = q[q0:q1, h].double(), k[k0:k1, h // share].double(), v[k0:k1, h // share].double()
            prod = Q @ K.T * scale
            add = torch.zeros_like(prod) if d2 is None else -slopes[h].double() * d2.double().sqrt() if bias is None else bias[:, h].double()[which]
            s = prod + add
            p = torch.softmax(s, 1)
            o = p @ V
            # a score: dim products and sums, scale, the bias (distance to 1 ulp, slope, log2 e), the sum, the running maximum and the
            # probability's exponent; all relative to the largest terms of the row
            # a score is off by dim + 8 half steps of its largest partial sums; a probability then by e^(2 of those) - 1, plus the
            # exponential's ulp and the sum over n keys (n half steps at most)
            ds_b = U32 * ((dim + 8) * (Q.abs() @ K.abs().T * scale) + 8 * add.abs() + 4 * s.abs().amax(1, keepdim=True))
            rel = 2 * ds_b.amax(1, keepdim=True) + U32 * (8 + 2 * math.sqrt(k1 - k0) * 4)
            pv = p @ V.abs()
            o_b = (rel + uP) * pv + U32 * (k1 - k0) ** 0.5 * 4 * pv
            val["out"][q0:q1, h] = o
            bnd["out"][q0:q1, h] = o_b + uT * (o.abs() + o_b)
            if go is None:
                continue
            G = go[q0:q1, h].double()
            dp, delta = G @ V.T, (G * o).sum(1, keepdim=True)
            # (the unrounded output still carries the rounded probabilities)
            delta_b = (G.abs() * o_b).sum(1, keepdim=True) + U32 * (dim + 2) * (G * o).abs().sum(1, keepdim=True)
            dp_b = U32 * (dim + 2) * (G.abs() @ V.abs().T)
            ds = p * (dp - delta)
            e = p * ((rel + 2 * U32) * (dp - delta).abs() + dp_b + delta_b + U32 * (dp.abs() + delta.abs()))
            er = e + uP * (ds.abs() + e)
            rows, cols = 4 * U32 * math.sqrt(k1 - k0), 4 * U32 * math.sqrt(q1 - q0)
            dq = ds @ K * scale
            dq_b = (er @ K.abs() + rows * (ds.abs() @ K.abs())) * scale + 2 * U32 * dq.abs()
            val["dq"][q0:q1, h], bnd["dq"][q0:q1, h] = dq, dq_b + uT * (dq.abs() + dq_b)
            val["dk"][k0:k1, h // share] += ds.T @ Q * scale
            bnd["dk"][k0:k1, h // share] += (er.T @ Q.abs() + cols * (ds.abs().T @ Q.abs())) * scale
            val["dv"][k0:k1, h // share] += p.T @ G
            bnd["dv"][k0:k1, h // share] += ((rel.T + uP + cols) * p.T) @ G.abs()
            if bias is not None:
                val["dt"][:, h] += torch.bincount(which.reshape(-1), ds.reshape(-1), minlength=bias.shape[0])
                n = max(q1 - q0, 1) * (k1 - k0)
                bnd["dt"][:, h] += torch.bincount(which.reshape(-1), (e + 4 * U32 * math.sqrt(n) * ds.abs()).reshape(-1), minlength=bias.shape[0])
    for name in ("dk", "dv"):
        bnd[name] += uT * (val[name].abs() + bnd[name])
    bnd["dt"] += U32 * val["dt"].abs()
    return val, bnd


def assert_within(got, val, bnd, floor, what):
    """|got - val| <= bnd + floor everywhere (floor: the type's smallest steps near zero)."""
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - val).abs() - bnd - floor
    worst = off.max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3e} beyond its bound (largest error {(got - val).abs().max().item():.3e})"


# -- the operators as differentiable 64-bit torch code, with ops' signatures (stand-ins inside a model) ---------------------------------------
def plain_group_norm(x, num_groups, weight=None, bias=None, segments=None, eps=1e-5, activation=None):
    out = torch.zeros_like(x, dtype=torch.float64)
    for lo, hi in [(0, x.shape[0])] if segments is None else segments.tolist():
        if hi <= lo:
            continue
        g = x[lo:hi].double().reshape(hi - lo, num_groups, -1)
        z = ((g - g.mean((0, 2), keepdim=True)) / torch.sqrt(g.var((0, 2), unbiased=False, keepdim=True) + eps)).flatten(1)
        z = z * (1 if weight is None else weight.double()) + (0 if bias is None else bias.double())
        rows = torch.arange(lo, hi, device=x.device)
        out = out.index_copy(0, rows, {None: z, "relu": z.relu(), "silu": z * torch.sigmoid(z)}[activation])
    return out.to(x.dtype)


def plain_segment_attention(q, k, v, seg_q=None, seg_k=None, *, coords_q=None, coords_k=None, slopes=None, bias=None, edges=None, scale=None):
    heads, share = q.shape[1], q.shape[1] // k.shape[1]
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for (q0, q1), (k0, k1) in zip([(0, q.shape[0])] if seg_q is None else seg_q.tolist(), [(0, k.shape[0])] if seg_k is None else seg_k.tolist()):
        if q1 <= q0 or k1 <= k0:
            continue
        Q, K, V = (t.double().transpose(0, 1).contiguous() for t in (q[q0:q1], k[k0:k1].repeat_interleave(share, 1), v[k0:k1].repeat_interleave(share, 1)))
        s = torch.matmul(Q, K.transpose(1, 2).contiguous()) * scale
        if slopes is not None or bias is not None:
            d2 = distance2(coords_q[q0:q1], coords_k[k0:k1])
            if slopes is not None:
                s = s - slopes.double()[:, None, None] * d2.double().sqrt()
            else:
                s = s + bias.double()[torch.bucketize(d2, torch.tensor(edges, dtype=torch.int64, device=q.device), right=True)].permute(2, 0, 1)
        o = torch.matmul(torch.softmax(s, 2), V).transpose(0, 1)
        out = out.index_copy(0, torch.arange(q0, q1, device=q.device), o)
    return out.to(q.dtype)
