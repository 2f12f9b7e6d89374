"""The scan-wise operators at the edges: large finite values beside a scan, scores and table entries far out, means far from zero (MI355X, against
64-bit forms; helpers and bounds of scanwise_ref)."""
import math

import pytest
import torch

from scanwise_ref import U32, assert_within, attention_ref, group_norm_ref, ranges
from test_gpu_scanwise import BF16, F16, F32, TINY, edges_of, generator, rand, voxel_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(device):
    from lidiff_amd import ops
    return ops


def attend(ops, q, k, v, go, *segments, bias=None, **kw):
    """Output and gradients of one call."""
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v) + (() if bias is None else (bias,))]
    out = ops.segment_attention(*leaves[:3], *segments, **kw, **({} if bias is None else {"bias": leaves[3]}))
    return (out.detach(),) + torch.autograd.grad(out, leaves, go)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("share", [1, 2])
def test_large_finite_values_beside_a_scan_change_no_bit_of_it(ops, dtype, share):
    """Another scan's rows and rows of no scan at 100 ... 60 000, in the values, the output's gradient, queries and keys."""
    gen = generator(31)
    seg, m = ranges([70, 50, 40], [3, 0, 2]).cuda(), 170
    q, go = rand(gen, m, 4, 32, dtype=dtype), rand(gen, m, 4, 32, dtype=dtype)
    k, v = rand(gen, m, 4 // share, 32, dtype=dtype), rand(gen, m, 4 // share, 32, dtype=dtype)
    kw = dict(coords_q=voxel_rows(gen, m), coords_k=voxel_rows(gen, m), bias=rand(gen, 8, 4), edges=edges_of(ops, 8))
    clean = attend(ops, q, k, v, go, seg, seg, **kw)
    for big in (1e2, 1e4, 6e4):
        q2, k2, v2, go2 = (t.clone() for t in (q, k, v, go))
        for t in (v2, go2, q2, k2):
            t[73:123], t[:3], t[123:125], t[165:] = big, big, big, big
        for name, got, want in zip(("out", "dq", "dk", "dv"), attend(ops, q2, k2, v2, go2, seg, seg, **kw), clean):
            assert torch.equal(got[3:73], want[3:73]) and torch.equal(got[125:165], want[125:165]), (name, big)


@pytest.mark.parametrize("bias", [None, 8])
def test_fp16_score_gradients_of_every_size(ops, bias):
    """Gradients of rows that differ by 10^8 in size, and masked keys with values near fp16's end: each key's and query's sum keeps the bits
    its own terms have."""
    gen = generator(32)
    nq, nk, h, d = 300, 400, 2, 32
    q, k, v = rand(gen, nq, h, d, dtype=F16), rand(gen, nk, h, d, dtype=F16), rand(gen, nk, h, d, dtype=F16)
    go = (rand(gen, nq, h, d) * 10.0 ** torch.randint(-4, 5, (nq, 1, 1), generator=gen, device="cuda")).clamp(-6e4, 6e4).to(F16)
    kw = {}
    if bias:
        ck, cq = voxel_rows(gen, nk), voxel_rows(gen, nq)
        ck[::7, 1] = 30000                                   # every seventh key is far away, in the last bucket: masked, its values huge
        v[::7] = 6e4
        table = rand(gen, bias, h)
        table[-1] = -math.inf
        cq[:, 1:] = cq[:, 1:].clamp(-200, 200)
        kw = dict(coords_q=cq, coords_k=ck, bias=table, edges=edges_of(ops, bias))
    got = attend(ops, q, k, v, go, **kw)
    # the 64-bit form without the masked keys (its bounds do not hold infinities); no other pair is in the last bucket
    seen = torch.arange(nk, device="cuda") % 7 != 0 if bias else torch.ones(nk, dtype=torch.bool, device="cuda")
    ref = {}
    if bias:
        ref = dict(cq=cq, ck=ck[seen], bias=table.nan_to_num(neginf=0.0), edges=kw["edges"])
        assert (cq[:, None, 1:] - ck[None, seen, 1:]).long().square().sum(-1).max() < kw["edges"][-1]
    val, bnd = attention_ref(q, k[seen], v[seen], go=go, **ref)
    for name, g in zip(("out", "dq", "dk", "dv"), (got[0], got[1], got[2][seen], got[3][seen])):
        assert_within(g, val[name], bnd[name], TINY[F16], f"{name} {bias}")
    if bias:
        assert (got[2][::7] == 0).all() and (got[3][::7] == 0).all()
    # small gradients alone: below fp16's normal range before they are lifted
    tiny = attend(ops, q, k, v, (rand(gen, nq, h, d) * 1e-3).to(F16), **kw)
    assert tiny[1].abs().max() > 0 and tiny[2].abs().max() > 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("entry", [math.inf, math.nan, -math.inf])
def test_a_bucket_that_no_pair_meets_has_no_gradient(ops, dtype, entry):
    """Whatever its entry holds: the places of a workgroup's tile without a query, or without a key, meet no bucket of their own."""
    gen = generator(33)
    for heads in (1, 2, 4):
        for nq, nk in ((5, 40), (70, 33), (128, 64)):
            q, k, v, go = (rand(gen, n, heads, 32, dtype=dtype) for n in (nq, nk, nk, nq))
            cq, ck = (torch.zeros(n, 4, dtype=torch.int32, device="cuda") for n in (nq, nk))
            cq[:, 1], ck[:, 1] = 1000, 1000 + torch.arange(nk, device="cuda")          # (far from the origin, near each other)
            table = rand(gen, 3, heads)
            table[2] = entry
            got = attend(ops, q, k, v, go, bias=table, edges=(400, 10000), coords_q=cq, coords_k=ck)
            val, bnd = attention_ref(q, k, v, go=go, bias=table.nan_to_num(0.0, 0.0, 0.0), edges=(400, 10000), cq=cq, ck=ck)
            assert (got[4][2] == 0).all()
            for name, g in zip(("out", "dq", "dk", "dv", "dt"), got):
                assert_within(g, val[name], bnd[name], 1e-30 if name == "dt" else TINY[dtype], f"{name} {heads} {nq}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("power", [5, 10, 14, 18, 20, 22, 23, 24, 28])
@pytest.mark.parametrize("sign", [1, -1])
def test_gradients_of_equal_scores_far_from_zero(ops, dtype, power, sign):
    """Keys with one and the same score of +-2^power (in units of log 2): the rebuilt probabilities are 1 / keys whatever the score is.

    The 64-bit form takes the scores 2^-power times as large: the same softmax, and its bounds then count the roundings of everything but the
    (equal) scores; dq and dk carry the scale as a factor.  All factors are powers of two."""
    gen = generator(34)
    for nk, heads, table in ((13, 2, False), (13, 2, True), (1300, 4, False), (1300, 1, True)):
        nq, d = 20, 32
        q, k = rand(gen, nq, heads, d, dtype=dtype), torch.zeros(nk, heads, d, dtype=dtype, device="cuda")
        q[..., 0], k[..., 0] = 2.0 ** (power // 2 - 1), sign * 2.0 ** (power - power // 2 - 1)
        v, go = rand(gen, nk, heads, d, dtype=dtype), rand(gen, nq, heads, d, dtype=dtype)
        kw = {}
        if table:
            c = lambda n: torch.zeros(n, 4, dtype=torch.int32, device="cuda")
            kw = dict(bias=torch.zeros(1, heads, device="cuda"), edges=(), coords_q=c(nq), coords_k=c(nk))
        scale = 4 * math.log(2)
        got = attend(ops, q, k, v, go, scale=scale, **kw)
        val, bnd = attention_ref(q, k, v, go=go, scale=scale * 2.0 ** -power, **{{"coords_q": "cq", "coords_k": "ck"}.get(n, n): t for n, t in kw.items()})
        for name, g in zip(("out", "dq", "dk", "dv", "dt"), got):
            more = 2.0 ** power if name in ("dq", "dk") else 1.0
            within = (val[name].abs() + bnd[name]) * more < torch.finfo(g.dtype).max      # (fp16 at 2^28: a few values of dk are beyond its range)
            assert within.all() or (dtype == F16 and power == 28 and name == "dk")
            assert_within(g[within], val[name][within] * more, bnd[name][within] * more, 1e-30 if name == "dt" else TINY[dtype], f"{name} {nk} {heads}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_table_entries_far_out_keep_their_order(ops, dtype):
    """Entries thousands to 10^38 apart: each key alone in its bucket, every pair of them visible to a query of its own -- the larger entry takes
    everything.  (Some stand within fp32's steps of each other's size, none of them equal.)"""
    for entries in ([-20000.0, -30000.0], [20000.0, 30000.0], [0.5, -1e4, -65504.0, torch.finfo(F32).min], [-1e9, -2e9, -3e38], [3e38, 1e38, 12000.0, 11000.0, -50.0],
                    [-400.0 * i for i in range(48)], [-9000.0 * i * i for i in range(20)], [1e5, 2e5, -1e5, 0.0, 99000.0]):
        n = len(entries)
        edges = tuple(range(1, 30 * n, 30)[:n - 1]) if n <= 3 else ops.distance_edges(n, 100, 16)
        # key b at a distance just inside bucket b, alone on a line from every query
        at = torch.tensor([0] + [math.isqrt(e - 1) + 1 for e in edges], device="cuda")
        assert [sum(e <= a * a for e in edges) for a in at.tolist()] == list(range(n))
        ck = torch.zeros(n, 4, dtype=torch.int32, device="cuda")
        ck[:, 1] = at
        pairs = [(i, j) for i in range(n) for j in range(n) if i < j]
        seg_q = torch.tensor([[p, p + 1] for p in range(len(pairs))], dtype=torch.int32)
        keys = torch.tensor(pairs, device="cuda").reshape(-1)
        gen = generator(35)
        q, v, go = rand(gen, len(pairs), 2, 32, dtype=dtype), rand(gen, n, 2, 32, dtype=dtype)[keys], rand(gen, len(pairs), 2, 32, dtype=dtype)
        k = rand(gen, 2 * len(pairs), 2, 32, dtype=dtype)
        table = torch.tensor([[e, e] for e in entries], device="cuda")
        table[:, 1] -= 3.0 if max(map(abs, entries)) < 1e6 else 0.0
        cq = torch.zeros(len(pairs), 4, dtype=torch.int32, device="cuda")
        got = attend(ops, q, k, v, go, seg_q.cuda(), (2 * seg_q).cuda(), coords_q=cq, coords_k=ck[keys].contiguous(), bias=table, edges=edges)
        winner = torch.tensor([max(p, key=lambda b: entries[b]) for p in pairs], device="cuda")
        want = v.reshape(len(pairs), 2, 2, 32)[torch.arange(len(pairs), device="cuda"), (winner != keys.view(-1, 2)[:, 0]).long()]
        # one value times a probability of one: exact for 16-bit operands; fp32's three pieces meet again in six products, sums and the division, a
        # half step or a cut (two half steps) each
        off = (got[0].double() - want.double()).abs()
        assert (off <= (16 * U32 if dtype == F32 else 0.0) * want.double().abs()).all(), (entries, off.max().item())
        # (a probability of one: score gradients are zero but for the roundings of do . v against do . out, dim + 2 half steps of each addend)
        assert all(torch.isfinite(g).all() for g in got)
        assert (got[4].abs() <= 2 * 34 * U32 * (go.double() * want.double()).abs().sum((0, 2))).all()


@pytest.mark.parametrize("mean", [0.0, 1e3, -1e5, 3e6])
@pytest.mark.parametrize("act", [None, "silu"])
def test_group_norm_of_means_far_from_zero(ops, mean, act):
    """Means up to 3 10^6 times the spread: errors are those of the spread.

    y: x - mean (the leading float: exact or a half step, the rest of it folded into the shift), rstd, the product and the shift, a half step
    each of at most 1 + |z|; silu as group_norm_ref counts it.  dx = rstd (t - ma - xh mb), each term off by a few half steps of itself and of
    mean |t xh|."""
    gen = generator(36)
    seg = ranges([3000, 1, 1000], [0, 2, 0]).cuda()
    x = rand(gen, 4003, 16) + mean
    x[5] += 50.0 * rand(gen, 16)
    dy = rand(gen, 4003, 16)
    val, _ = group_norm_ref(x, 4, None, None, seg, 1e-5, act, dy)
    plain, _ = group_norm_ref(x, 4, None, None, seg, 1e-5, None, dy)
    z = plain["y"].abs()
    leaf = x.clone().requires_grad_()
    y = ops.group_norm(leaf, 4, segments=seg, activation=act)
    dx, = torch.autograd.grad(y, [leaf], dy)
    assert_within(y.detach(), val["y"], 16 * U32 * (1 + z) * (1 + (z if act else 0)), 0, f"y {mean}")
    for lo, hi in seg.tolist():
        rstd = (x[lo:hi].double().reshape(hi - lo, 4, 4).var((0, 2), unbiased=False) + 1e-5).rsqrt().repeat_interleave(4)
        t = 1.1 * dy[lo:hi].double().abs()
        size = t + t.mean() * 8 + z[lo:hi] * (t * (1 + z[lo:hi])).mean() * 8
        assert_within(dx[lo:hi], val["dx"][lo:hi], 32 * U32 * rstd * size * (1 + (z[lo:hi] if act else 0)), 0, f"dx {mean}")


def test_index_tensors_at_any_offset_of_their_storage(ops):
    """Segments and coordinates that are views one element into a buffer: the results of aligned copies."""
    gen = generator(37)
    x, c, seg = rand(gen, 90, 32), voxel_rows(gen, 90), ranges([50, 0, 40]).cuda()
    c[60:, 0] = 1
    def off(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)
    assert torch.equal(ops.group_norm(x, 8, segments=off(seg)), ops.group_norm(x, 8, segments=seg))
    assert ops.batch_segments(off(c)).tolist() == [[0, 60], [60, 90]]
    q, slopes = rand(gen, 90, 4, 32), torch.full((4,), 0.02, device="cuda")
    assert torch.equal(ops.segment_attention(q, q, q, off(seg), off(seg), coords_q=off(c), coords_k=off(c), slopes=off(slopes)),
                       ops.segment_attention(q, q, q, seg, seg, coords_q=c, coords_k=c, slopes=slopes))


def test_offsets_beyond_32_bits(ops):
    """Row matrices of more than 2^31 elements, keys whose rows stand 8 MiB apart: the last rows' results are those of a copy of them."""
    gen = generator(38)
    rows, c = 8_600_000, 256
    x = torch.empty(rows, c, dtype=BF16, device="cuda")
    x[:-1000] = 3.0
    x[-1000:] = rand(gen, 1000, c, dtype=BF16)
    seg = torch.tensor([[0, rows - 1000], [rows - 1000, rows]], dtype=torch.int32, device="cuda")
    leaf, last = x.requires_grad_(), x[-1000:].detach().clone().requires_grad_()
    y = ops.group_norm(leaf, 8, segments=seg, activation="silu")
    z = ops.group_norm(last, 8, activation="silu")
    # (more slabs share the rows of a scan alone: the doubles' sums round elsewhere, 2^-24 of the statistics at most, a half step of bf16 once)
    assert ((y[-1000:].double() - z.double()).abs() <= 2.0 ** -7 * z.double().abs() + 1e-6).all() and (y[:1000] == 0).all()
    go = rand(gen, 1000, c, dtype=BF16)
    dy = torch.zeros_like(x)
    dy[-1000:] = go
    g, = torch.autograd.grad(y, [leaf], dy)
    h, = torch.autograd.grad(z, [last], go)
    assert ((g[-1000:].double() - h.double()).abs() <= 2.0 ** -7 * h.double().abs() + 1e-5).all() and (g[:1000] == 0).all()
    del x, y, g, dy, leaf
    torch.cuda.empty_cache()
    wide = torch.empty(600, (1 << 22) - 8, dtype=BF16, device="cuda")
    parts = [rand(gen, 600, 2, 32, dtype=BF16) for _ in range(3)]
    for i, t in enumerate(parts):
        wide[:, 64 * i:64 * i + 64] = t.reshape(600, 64)
    slots = [wide[:, 64 * i:64 * i + 64].unflatten(1, (2, 32)) for i in range(3)]
    go, slopes, cs = rand(gen, 600, 2, 32, dtype=BF16), torch.full((2,), 0.02, device="cuda"), voxel_rows(gen, 600)
    outs = []
    for q, k, v in (slots, parts):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        assert leaves[0].stride(0) in ((1 << 22) - 8, 64)
        out = ops.segment_attention(*leaves, coords_q=cs, coords_k=cs, slopes=slopes)
        outs.append((out.detach(),) + torch.autograd.grad(out, leaves, go))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bias", ["none", "slopes", 16])
def test_few_keys_are_weighted_with_more_than_the_operands_bits(ops, dtype, bias):
    """Up to a tile of keys a scan, 16-bit operands: the output is off by its own rounding (and 2^-15 of the weighted values' sizes: two pieces of
    bf16 hold 16 bits), dq and dk by the score gradients' rounding and their own -- do . out brings none of the probabilities'."""
    gen = generator(39)
    heads, lens_q, lens_k = 4, [150, 12, 1, 60], [2, 64, 3, 0]
    seg_q, seg_k = ranges(lens_q), ranges(lens_k)
    mq, mk = sum(lens_q), sum(lens_k)
    q, k, v, go = (rand(gen, n, heads, 32, dtype=dtype) for n in (mq, mk, mk, mq))
    kw = {} if bias == "none" else dict(coords_q=voxel_rows(gen, mq), coords_k=voxel_rows(gen, mk))
    if bias == "slopes":
        kw["slopes"] = torch.full((heads,), 0.01, device="cuda")
    elif bias != "none":
        kw.update(bias=rand(gen, bias, heads), edges=edges_of(ops, bias))
    got = attend(ops, q, k, v, go, seg_q.cuda(), seg_k.cuda(), **kw)
    names = {"coords_q": "cq", "coords_k": "ck"}
    # the 64-bit form on fp32 copies of the operands: its bounds then count no rounding of probabilities or score gradients
    val, bnd = attention_ref(q.float(), k.float(), v.float(), seg_q, seg_k, go=go.float(), **{names.get(n, n): t for n, t in kw.items()})
    u = torch.finfo(dtype).eps / 2
    size = torch.zeros_like(val["out"])
    for (q0, q1), (k0, k1) in zip(seg_q.tolist(), seg_k.tolist()):
        if k1 > k0:
            size[q0:q1] = v[k0:k1].double().abs().amax(0)
    assert_within(got[0], val["out"], bnd["out"] + 2.0 ** -15 * size + u * (val["out"].abs() + size * 2.0 ** -14), TINY[dtype], "out")
    for name, g in (("dq", got[1]), ("dk", got[2]), ("dv", got[3])):
        # (2-norms: independent roundings of the terms, of the sums, of the result: root of two half steps' mean squares, u / sqrt(3) each at
        # most, a fifth on top for the few terms there are)
        off = (g.double() - val[name]).norm() / val[name].norm()
        assert off <= 1.2 * math.sqrt(2 / 3) * u + 1e-5, (name, off.item() / u)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bias", ["none", "slopes", 16])
def test_a_lone_key_has_no_score_gradients(ops, dtype, bias):
    """Scans of one key: its probability is 1, so the output is its value and dq, dk and the table's gradient are zero, not roundings."""
    gen = generator(40)
    lens_q, lens_k = [200, 3, 0, 1, 70], [1, 1, 1, 1, 5]
    seg_q, seg_k = ranges(lens_q, [2, 0, 0, 0, 1]), ranges(lens_k, [1, 0, 3, 0, 0])
    mq, mk = int(seg_q[-1, 1]), int(seg_k[-1, 1])
    q, k, v, go = (rand(gen, n, h, 32, dtype=dtype) for n, h in ((mq, 4), (mk, 2), (mk, 2), (mq, 4)))
    kw = {} if bias == "none" else dict(coords_q=voxel_rows(gen, mq), coords_k=voxel_rows(gen, mk))
    if bias == "slopes":
        kw["slopes"] = torch.full((4,), 0.01, device="cuda")
    elif bias != "none":
        kw.update(bias=rand(gen, bias, 4), edges=edges_of(ops, bias))
    got = attend(ops, q, k, v, go, seg_q.cuda(), seg_k.cuda(), **kw)
    val, bnd = attention_ref(q, k, v, seg_q, seg_k, go=go, **{{"coords_q": "cq", "coords_k": "ck"}.get(n, n): t for n, t in kw.items()})
    for name, g in zip(("out", "dq", "dk", "dv", "dt"), got):
        assert_within(g, val[name], bnd[name], 1e-30 if name == "dt" else TINY[dtype], name)
    assert (got[1][:int(seg_q[3, 1])] == 0).all() and (got[2][:int(seg_k[3, 1])] == 0).all()
    if bias == 16:
        one = attend(ops, q[:200], k[:1], v[:1], go[:200], **{n: t[:200 if n == "coords_q" else 1] if n[:6] == "coords" else t for n, t in kw.items()})
        assert (one[4] == 0).all()


@pytest.mark.parametrize("nq,nk,heads,kv_heads,dim", [(1, 8893, 2, 2, 128), (320, 6816, 4, 1, 64), (20000, 1500, 2, 2, 32)])
def test_fp32_gradients_of_long_sums(ops, nq, nk, heads, kv_heads, dim):
    """fp32 sums over thousands of rows: no further from 64 bits than the same formulas in fp32 torch operations (5 / 4 of their error), whose sums
    are pairwise -- the matrix pipe's one-sided cuts must not add up along a scan."""
    gen = generator(41)
    q, k, v, go = rand(gen, nq, heads, dim), rand(gen, nk, kv_heads, dim), rand(gen, nk, kv_heads, dim), rand(gen, nq, heads, dim)
    got = attend(ops, q, k, v, go)
    def formulas(dtype):
        res = [torch.zeros(t.shape, dtype=dtype, device="cuda") for t in (q, q, k, v)]
        for h in range(heads):
            Q, K, V, G = (t.to(dtype)[:, i].contiguous() for t, i in ((q, h), (k, h * kv_heads // heads), (v, h * kv_heads // heads), (go, h)))
            p = torch.softmax(Q @ K.T.contiguous() / math.sqrt(dim), 1)
            out = p @ V
            ds = p * (G @ V.T.contiguous() - (G * out).sum(1, keepdim=True))
            res[0][:, h], res[1][:, h] = out, ds @ K / math.sqrt(dim)
            res[2][:, h * kv_heads // heads] += ds.T.contiguous() @ Q / math.sqrt(dim)
            res[3][:, h * kv_heads // heads] += p.T.contiguous() @ G
        return res
    for name, mine, exact, plain in zip(("out", "dq", "dk", "dv"), got, formulas(torch.float64), formulas(F32)):
        off, other = ((t.double() - exact).norm().item() for t in (mine, plain))
        # (12 half steps of the result: six products with a cut each, scores and exponentials of a few half steps each; below that both are as good)
        assert off <= max(1.25 * other, 12 * U32 * exact.norm().item()), (name, off / exact.norm().item(), other / exact.norm().item())
