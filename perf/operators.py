"""What is measured of the scan-wise operators: group normalisation with an activation, and attention between the voxel rows of the
same scan whose scores carry a bias of distance (fixed slopes, or a learned table by distance buckets).

A batch of scans is ONE row matrix; `segments` [S, 2] holds the first row and the row behind the last one of every scan.  Sizes are
those of the denoiser's maps on a 180 000-point scan (voxel rows per tensor stride: 179 795 / 178 323 / 167 602 / 115 953 / 41 157
of the noisy cloud, 12 809 / 5 824 at strides 8 / 16 of the partial scan) at the training batch of two, down to windows of a few
voxels and the single row of a pooled query.

`own = False` computes the operators from elementary torch operations; `own = True` calls lidiff_amd.ops.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def lens(rows, scans, ragged):
    """Rows of each scan: the first has `rows`, the others down to (1 - ragged) of it; with ragged = 1 some scans are empty."""
    return [0 if ragged == 1 and i % 11 == 10 else max(1, round(rows * (1 - ragged * ((37 * i) % 100) / 100))) for i in range(scans)]


def squared_edges(buckets, stride, reach):
    """Squared distances at which the next bucket begins: one bucket per voxel of the map's stride in the first half, then evenly in
    the logarithm up to `reach` voxels."""
    near = buckets // 2
    far = [near * (reach / near) ** (i / (buckets - 1 - near)) for i in range(1, buckets - near)]
    return tuple(math.ceil((stride * r) ** 2) for r in [float(i) for i in range(1, near + 1)] + far)


def listed():
    norm = dict(op="norm", eps=1e-5)
    dist = dict(op="attention", buckets=0, stride=16, reach=0)
    table = dict(op="attention", buckets=32, stride=16, reach=100)
    return [
        # the denoiser's condition latent of one scan at inference: a call of a few microseconds, latency counts
        dict(norm, name="norm_latent", rows=5824, scans=1, ragged=0.0, channels=256, groups=32, act="silu", dtype="f32", train=False),
        # the stem of a training step: 32 channels of every voxel of two scans
        dict(norm, name="norm_stem_train", rows=179795, scans=2, ragged=0.1, channels=32, groups=8, act="silu", dtype="f32", train=True),
        # stride 8 of a bf16 training step
        dict(norm, name="norm_stride8_train_bf16", rows=115953, scans=2, ragged=0.1, channels=256, groups=32, act="relu", dtype="bf16", train=True),
        # windows of a few voxels, each normalised by itself, some of them empty
        dict(norm, name="norm_windows_train_f16", rows=301, scans=96, ragged=1.0, channels=96, groups=12, act="none", dtype="f16", train=True),
        # one pooled row per scan reads its scan's latent: the single-row form
        dict(dist, name="pool_one_row", q_rows=1, k_rows=5824, scans=2, ragged=0.1, heads=8, kv_heads=8, dim=32, dtype="bf16", train=False),
        # self-attention of the condition latent, full precision, inference
        dict(dist, name="latent_self_f32", q_rows=5824, k_rows=5824, scans=1, ragged=0.0, heads=8, kv_heads=8, dim=32, dtype="f32", train=False),
        # windows of a few voxels, some of them without keys, shared key heads, training
        dict(dist, name="windows_train_f16", q_rows=301, k_rows=283, scans=96, ragged=1.0, heads=4, kv_heads=2, dim=64, dtype="f16", train=True),
        # the noisy cloud at stride 16 reads the partial scan's latent, training batch of two
        dict(dist, name="cross_train_bf16", q_rows=41157, k_rows=5824, scans=2, ragged=0.1, heads=8, kv_heads=8, dim=32, dtype="bf16", train=True),
        # a handful of pooled rows with the learned bias
        dict(table, name="pool_rows_table", q_rows=13, k_rows=5824, scans=2, ragged=0.1, heads=8, kv_heads=8, dim=32, dtype="f32", train=False),
        # the guidance pair of a denoising step: two replicas of the noisy cloud read the latent
        dict(table, name="cross_table_bf16", q_rows=41157, k_rows=5824, scans=2, ragged=0.0, heads=8, kv_heads=8, dim=32, dtype="bf16", train=False),
        # a late, denoised cloud reads the latent, full precision, training
        dict(table, name="cross_table_train_f32", q_rows=7702, k_rows=5824, scans=2, ragged=0.1, heads=4, kv_heads=4, dim=64, dtype="f32", train=True),
        # self-attention of the partial scan at stride 8, training: the largest
        dict(table, name="self_table_train_bf16", q_rows=12809, k_rows=12809, scans=2, ragged=0.1, heads=8, kv_heads=8, dim=32, dtype="bf16", train=True,
             stride=8, reach=200),
    ]


def draw(rng):
    log = lambda lo, hi: max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    scans, ragged = rng.choice([(1, 0.0), (2, 0.1), (2, 0.5), (5, 0.5), (24, 1.0), (96, 1.0)])
    dtype, train = rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.6
    if rng.random() < 0.4:
        channels, groups = rng.choice([(32, 8), (64, 8), (96, 12), (96, 32), (128, 32), (256, 32), (256, 1), (48, 16), (20, 4)])
        return dict(op="norm", eps=1e-5, rows=log(1, min(180000, 40_000_000 // (scans * channels))), scans=scans, ragged=ragged, channels=channels, groups=groups,
                    act=rng.choice(["none", "relu", "silu"]), dtype=dtype, train=train)
    heads, kv_heads, dim = rng.choice([(8, 8, 32), (8, 2, 32), (4, 4, 64), (4, 1, 64), (2, 2, 128), (3, 3, 32), (6, 2, 16), (4, 4, 24), (1, 1, 96)])
    k_rows = log(1, 12000 if scans <= 2 else 4000 if scans <= 5 else 400)
    q_rows = log(1, min(41000, 230_000_000 // (scans * k_rows * (2 if dtype == "f32" else 1) * max(1, heads * dim // 256))) if scans <= 5 else 400)
    buckets = rng.choice([0, 0, 16, 32, 48])
    return dict(op="attention", buckets=buckets, stride=rng.choice([4, 8, 16]), reach=rng.choice([60, 100, 120]) if buckets else 0, q_rows=q_rows, k_rows=k_rows,
                scans=scans, ragged=ragged, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, train=train)


def _segments(lengths):
    ends = torch.tensor(lengths, dtype=torch.int64).cumsum(0)
    return torch.stack([ends - torch.tensor(lengths, dtype=torch.int64), ends], 1).to(torch.int32).cuda()


def _coords(lengths, stride, gen):
    """Voxel coordinates (batch, x, y, z) of scans as a sensor on the ground sees them, on the map's lattice."""
    m = sum(lengths)
    p = torch.randn(m, 3, generator=gen, device="cuda") * torch.tensor([300.0, 300.0, 24.0], device="cuda")
    b = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).cuda()
    return torch.cat([b[:, None], (torch.floor(p / stride) * stride).long()], 1).to(torch.int32).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    if case["op"] == "norm":
        n = lens(case["rows"], case["scans"], case["ragged"])
        c = case["channels"]
        # features behind a convolution: channels with means and spreads of their own
        x = (rnd(sum(n), c) * (0.5 + rnd(c).abs()) + rnd(c)).to(dtype)
        return dict(case=case, lens=n, seg=_segments(n), x=x, weight=1 + 0.1 * rnd(c), bias=0.1 * rnd(c), dy=rnd(sum(n), c).to(dtype) if case["train"] else None)
    nq, nk = (lens(case[k], case["scans"], case["ragged"]) for k in ("q_rows", "k_rows"))
    if case["q_rows"] == case["k_rows"]:
        nk = nq
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    s = dict(case=case, lens_q=nq, lens_k=nk, seg_q=_segments(nq), seg_k=_segments(nk), q=rnd(sum(nq), h, d).to(dtype), k=rnd(sum(nk), hk, d).to(dtype),
             v=rnd(sum(nk), hk, d).to(dtype), coords_q=_coords(nq, case["stride"], gen), coords_k=_coords(nk, case["stride"], gen),
             do=rnd(sum(nq), h, d).to(dtype) if case["train"] else None)
    if case["q_rows"] == case["k_rows"]:
        s["coords_k"] = s["coords_q"]
    if case["buckets"]:
        s["edges"], s["table"] = squared_edges(case["buckets"], case["stride"], case["reach"]), 0.5 * rnd(case["buckets"], h)
    else:
        # slopes of a geometric series over the heads, per voxel of the map's stride
        s["slopes"] = (2.0 ** (-torch.arange(1, h + 1, device="cuda") * 8 / h) / case["stride"]).float()
    return s


def _padding(lengths, device):
    """[S, L] row index of every scan's rows (0 behind its end) and the mask of the real ones."""
    n = torch.tensor(lengths, device=device)
    at = torch.arange(max(max(lengths), 1), device=device)
    real = at < n[:, None]
    return torch.where(real, (n.cumsum(0) - n)[:, None] + at, 0), real


def _plain_norm(x, weight, bias, lengths, groups, eps, act):
    rows, real = _padding(lengths, x.device)
    keep = real[:, :, None, None]
    p = x.float()[rows].reshape(*rows.shape, groups, -1)
    count = (real.sum(1) * p.shape[-1]).clamp(min=1)[:, None, None, None]
    mean = torch.where(keep, p, 0).sum((1, 3), keepdim=True) / count
    off = torch.where(keep, p - mean, 0)
    var = (off * off).sum((1, 3), keepdim=True) / count
    z = (off / torch.sqrt(var + eps)).flatten(2)[real] * weight + bias
    return (z if act == "none" else z.clamp(min=0) if act == "relu" else z / (1 + torch.exp(-z))).to(x.dtype)


def _plain_attention(s, q, k, v, table):
    case = s["case"]
    share = case["heads"] // case["kv_heads"]
    rq, real_q = _padding(s["lens_q"], q.device)
    rk, real_k = _padding(s["lens_k"], q.device)
    qp = q.float()[rq].transpose(1, 2)
    kp, vp = (t.float()[rk].repeat_interleave(share, 2).transpose(1, 2) for t in (k, v))
    apart = s["coords_q"][rq][:, :, None, 1:].float() - s["coords_k"][rk][:, None, :, 1:].float()
    d2 = (apart * apart).sum(-1)
    if table is not None:
        bucket = torch.bucketize(d2, torch.tensor(s["edges"], device=q.device).float(), right=True, out_int32=True)
        chosen = (bucket[..., None] == torch.arange(table.shape[0], device=q.device, dtype=torch.int32)).float()
        # (a product per query row: the gradient's long sum over all pairs is then taken row by row)
        bias = (chosen @ table.expand(*chosen.shape[:2], *table.shape)).permute(0, 3, 1, 2)
    else:
        bias = -s["slopes"][:, None, None] * torch.sqrt(d2)[:, None]
    score = torch.where(real_k[:, None, None], (qp @ kp.transpose(2, 3)) / math.sqrt(case["dim"]) + bias, -torch.inf)
    e = torch.exp(score - score.amax(3, keepdim=True).detach().clamp(min=-3e38))
    out = (e @ vp) / e.sum(3, keepdim=True).clamp(min=1e-30)
    return out.transpose(1, 2)[real_q].to(q.dtype)


def run(state):
    case = state["case"]
    train = case["train"]
    leaf = (lambda t: t.detach().requires_grad_()) if train else (lambda t: t)
    if case["op"] == "norm":
        x, w, b = leaf(state["x"]), leaf(state["weight"]), leaf(state["bias"])
        if own:
            from lidiff_amd import ops
            y = ops.group_norm(x, case["groups"], w, b, segments=state["seg"], eps=case["eps"], activation=None if case["act"] == "none" else case["act"])
        else:
            y = _plain_norm(x, w, b, state["lens"], case["groups"], case["eps"], case["act"])
        if not train:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), state["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    q, k, v = leaf(state["q"]), leaf(state["k"]), leaf(state["v"])
    table = leaf(state["table"]) if case["buckets"] else None
    if own:
        from lidiff_amd import ops
        out = ops.segment_attention(q, k, v, state["seg_q"], state["seg_k"], coords_q=state["coords_q"], coords_k=state["coords_k"],
                                    slopes=state.get("slopes"), bias=table, edges=state.get("edges"))
    else:
        out = _plain_attention(state, q, k, v, table)
    if not train:
        return {"out": out}
    grads = torch.autograd.grad(out, (q, k, v) + (() if table is None else (table,)), state["do"])
    return {"out": out.detach(), **dict(zip(("dq", "dk", "dv", "dtable"), grads))}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n, c = sum(lens(case["rows"], case["scans"], case["ragged"])), case["channels"]
        passes = 4 if case["train"] else 2          # x -> y; and dy -> dx (x is there already)
        return {"bytes": passes * n * c * size + 4 * c * (4 if case["train"] else 2) + 8 * case["scans"], "flops": n * c * (30 if case["train"] else 12)}
    nq, nk = (lens(case[k], case["scans"], case["ragged"]) for k in ("q_rows", "k_rows"))
    if case["q_rows"] == case["k_rows"]:
        nk = nq
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    pairs = sum(a * b for a, b in zip(nq, nk))
    mq, mk = sum(nq), sum(nk)
    sweep = size * d * (2 * h * mq + 2 * hk * mk)                  # q, out and k, v; their gradients once more
    return {"bytes": sweep * (2 if case["train"] else 1) + 16 * (mq + mk) + 16 * case["scans"] + 4 * case["buckets"] * h * (2 if case["train"] else 1),
            "flops": pairs * h * d * 2 * (7 if case["train"] else 2)}


def exact(case, seed):
    """In 64 bits, scan by scan (and query block by query block), gradients by their formulas."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        g, c = case["groups"], case["channels"]
        ys, dxs = [], []
        dw = db = torch.zeros(c, dtype=torch.float64, device="cuda")
        w, b = s["weight"].double(), s["bias"].double()
        for x, dy in zip(s["x"].double().split(s["lens"]), (s["x"] if s["dy"] is None else s["dy"]).double().split(s["lens"])):
            if not len(x):
                ys.append(x)
                dxs.append(x)
                continue
            var, mean = torch.var_mean(x.reshape(len(x), g, -1), dim=(0, 2), unbiased=False)
            rstd = (var + case["eps"]).rsqrt().repeat_interleave(c // g)
            xh = (x - mean.repeat_interleave(c // g)) * rstd
            z = xh * w + b
            sig = torch.sigmoid(z)
            slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": sig * (1 + z * (1 - sig))}[case["act"]]
            ys.append({"none": z, "relu": z.relu(), "silu": z * sig}[case["act"]])
            if case["train"]:
                dz = dy * slope
                dw, db = dw + (dz * xh).sum(0), db + dz.sum(0)
                t = (dz * w).reshape(len(x), g, -1)
                xg = xh.reshape(len(x), g, -1)
                dxs.append(((t - t.mean((0, 2), keepdim=True) - xg * (t * xg).mean((0, 2), keepdim=True)).flatten(1)) * rstd)
        return {"y": torch.cat(ys), "dx": torch.cat(dxs), "dweight": dw, "dbias": db} if case["train"] else {"y": torch.cat(ys)}
    share, scale = case["heads"] // case["kv_heads"], 1 / math.sqrt(case["dim"])
    out, dq = torch.zeros_like(s["q"], dtype=torch.float64), torch.zeros_like(s["q"], dtype=torch.float64)
    dk, dv = torch.zeros_like(s["k"], dtype=torch.float64), torch.zeros_like(s["v"], dtype=torch.float64)
    dt = torch.zeros(max(1, case["buckets"]), case["heads"], dtype=torch.float64, device="cuda")
    edges = torch.tensor(s.get("edges", ()), device="cuda", dtype=torch.int64)
    q0 = k0 = 0
    for nq, nk in zip(s["lens_q"], s["lens_k"]):
        for lo in range(q0, q0 + nq if nk else q0, 2048):
            rows, keys = slice(lo, min(q0 + nq, lo + 2048)), slice(k0, k0 + nk)
            d2 = (s["coords_q"][rows, None, 1:].long() - s["coords_k"][None, keys, 1:].long()).square().sum(-1)
            which = torch.bucketize(d2, edges, right=True) if case["buckets"] else None
            for h in range(case["heads"]):
                q, k, v = s["q"][rows, h].double(), s["k"][keys, h // share].double(), s["v"][keys, h // share].double()
                p = torch.softmax(q @ k.T * scale + (s["table"][:, h].double()[which] if case["buckets"] else -s["slopes"][h].double() * d2.double().sqrt()), 1)
                o = out[rows, h] = p @ v
                if case["train"]:
                    do = s["do"][rows, h].double()
                    ds = p * (do @ v.T - (do * o).sum(1, keepdim=True))
                    dq[rows, h] = ds @ k * scale
                    dk[keys, h // share] += ds.T @ q * scale
                    dv[keys, h // share] += p.T @ do
                    if case["buckets"]:
                        dt[:, h] += torch.bincount(which.reshape(-1), ds.reshape(-1), minlength=case["buckets"])
        q0, k0 = q0 + nq, k0 + nk
    if not case["train"]:
        return {"out": out}
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, **({"dtable": dt} if case["buckets"] else {})}
