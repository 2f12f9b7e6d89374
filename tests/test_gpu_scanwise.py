"""Group normalisation and attention within a scan (ops.group_norm, ops.segment_attention) on the MI355X against 64-bit forms."""
import math

import pytest
import torch

from scanwise_ref import assert_within, attention_ref, group_norm_ref, ranges

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TINY = {F32: 1e-30, BF16: 1e-30, F16: 2.0 ** -24}         # the smallest step near zero (fp16: its denormals' spacing)


@pytest.fixture(scope="module")
def ops(device):
    from lidiff_amd import ops
    return ops


def rand(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def voxel_rows(gen, m, stride=16, spread=200.0):
    c = (torch.randn(m, 3, generator=gen, device="cuda") * torch.tensor([spread, spread, spread / 8], device="cuda") / stride).floor().int() * stride
    return torch.cat([torch.zeros(m, 1, dtype=torch.int32, device="cuda"), c], 1).contiguous()


# -- group norm ---------------------------------------------------------------------------------------------------------------------
NORM_CASES = [
    # lengths, gaps, channels, groups
    ([1], None, 4, 1), ([1], None, 256, 32), ([2], None, 20, 5), ([63, 0, 1, 130], None, 32, 8), ([5, 700], [3, 2], 96, 12), ([1000], [0], 256, 1),
    ([257], None, 1024, 32), ([33, 31], [1, 0], 1020, 255), ([4000, 3333], None, 48, 16), ([7] * 90 + [0] * 10 + [1] * 30, None, 64, 8), ([0, 0], [5, 0], 8, 2),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("case", range(len(NORM_CASES)))
def test_group_norm_against_64_bits(ops, case, act, dtype):
    lengths, gaps, c, groups = NORM_CASES[case]
    gen = generator(100 + case)
    seg = ranges(lengths, gaps)
    m = int(seg[-1, 1]) + (4 if gaps else 0)                      # rows behind the last scan as well
    x = (rand(gen, m, c) * (0.5 + rand(gen, c).abs()) + 2 * rand(gen, c)).to(dtype)
    w, b, dy = 1 + 0.2 * rand(gen, c), 0.3 * rand(gen, c), rand(gen, m, c, dtype=dtype)
    val, _ = group_norm_ref(x, groups, w, b, seg, 1e-5, None)
    if act == "relu":                                             # no gradient where a rounding could flip the sign
        dy = torch.where(val["y"].abs() < 1e-3, 0, dy)
    val, bnd = group_norm_ref(x, groups, w, b, seg, 1e-5, act, dy)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = ops.group_norm(leaves[0], groups, leaves[1], leaves[2], segments=seg.cuda(), eps=1e-5, activation=act)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == F32
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert_within(got.detach(), val[name], bnd[name], TINY[dtype] if name in ("y", "dx") else 1e-30, f"{name} {NORM_CASES[case]} {act} {dtype}")
    outside = torch.ones(m, dtype=torch.bool)
    for lo, hi in seg.tolist():
        outside[lo:hi] = False
    assert (y[outside.cuda()] == 0).all() and (dx[outside.cuda()] == 0).all()
    again = ops.group_norm(x, groups, w, b, segments=seg.cuda(), eps=1e-5, activation=act)
    assert torch.equal(again, y)


def test_group_norm_without_affine_or_segments_and_any_layout(ops):
    gen = generator(1)
    x = rand(gen, 500, 64)
    val, bnd = group_norm_ref(x, 8, None, None, None, 1e-5, "silu")
    assert_within(ops.group_norm(x, 8, activation="silu"), val["y"], bnd["y"], 0, "no affine")
    wide = torch.zeros(500, 96, device="cuda")
    wide[:, 8:72] = x
    assert torch.equal(ops.group_norm(wide[:, 8:72], 8, activation="silu"), ops.group_norm(x, 8, activation="silu"))
    flat = torch.zeros(500 * 64 + 1, device="cuda")
    flat[1:] = x.reshape(-1)
    assert torch.equal(ops.group_norm(flat[1:].view(500, 64), 8, activation="silu"), ops.group_norm(x, 8, activation="silu"))
    assert ops.group_norm(x[:0], 8).shape == (0, 64)
    empty = x[:0].clone().requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(ops.group_norm(empty, 8, w).sum(), [empty, w])
    assert gx.shape == (0, 64) and (gw == 0).all()
    one = x[:1].expand(500, 64).detach().requires_grad_()             # a broadcast input: every row the same gradient shape
    g, = torch.autograd.grad(ops.group_norm(one, 8).sum(), [one])
    assert g.shape == (500, 64)


def test_group_norm_keeps_scans_apart(ops):
    """Inf and NaN of one scan stay there; a scan alone gives the bits it gives in a batch of the same size class."""
    gen = generator(2)
    x = rand(gen, 300, 32)
    seg = ranges([100, 100, 100]).cuda()
    clean = ops.group_norm(x, 8, segments=seg)
    bad = x.clone()
    bad[150, 3], bad[160, 9] = math.nan, math.inf
    got = ops.group_norm(bad, 8, segments=seg)
    assert torch.equal(got[:100], clean[:100]) and torch.equal(got[200:], clean[200:])
    assert torch.isnan(got[100:200, :4]).all() and torch.isnan(got[100:200, 8:12]).all()
    assert torch.equal(got[100:200, 12:], clean[100:200, 12:])
    leaf = bad.clone().requires_grad_()
    g, = torch.autograd.grad(ops.group_norm(leaf, 8, segments=seg, activation="silu"), [leaf], torch.ones_like(leaf))
    assert torch.isfinite(g[:100]).all() and torch.isfinite(g[200:]).all()


def test_group_norm_of_a_far_mean(ops):
    """Statistics in double: a mean 10^4 times the spread costs what the fp32 mean's own rounding costs."""
    gen = generator(3)
    x = rand(gen, 4000, 16) + 1e4
    val, bnd = group_norm_ref(x, 4, None, None, None, 1e-5, None)
    assert_within(ops.group_norm(x, 4), val["y"], bnd["y"], 0, "far mean")


# -- attention ----------------------------------------------------------------------------------------------------------------------
def edges_of(ops, buckets, stride=16):
    return ops.distance_edges(buckets, 100, stride) if buckets > 1 else ()


ATTENTION_CASES = [
    # query lengths, key lengths, gaps, H, Hkv, D, bias
    ([1], [1], None, 1, 1, 32, "none"), ([1], [700], None, 8, 8, 32, "slopes"), ([1, 1], [5824, 3000], None, 8, 8, 32, "slopes"),
    ([13, 1], [1000, 2300], None, 8, 8, 32, 32), ([17], [63], None, 4, 4, 32, "slopes"), ([64], [64], None, 4, 4, 32, 16), ([65, 128], [129, 64], None, 8, 2, 32, 32),
    ([40, 0, 30, 20], [10, 20, 0, 33], None, 4, 2, 64, "slopes"), ([100, 3], [90, 200], [2, 5], 2, 2, 64, 32), ([77], [150], None, 3, 3, 64, 7),
    ([50, 61], [70, 40], [0, 3], 2, 1, 128, 48), ([33], [200], None, 1, 1, 96, "none"), ([200], [130], [4], 6, 2, 16, "slopes"), ([90], [90], None, 4, 4, 24, 2),
    ([55, 200], [80, 300], None, 4, 1, 8, 1), ([9] * 70 + [1] * 9, [5] * 70 + [130] * 9, None, 4, 4, 32, 16), ([30], [0], None, 2, 2, 32, "slopes"),
    ([500, 300], [900, 1100], None, 12, 3, 32, 32), ([3000], [70], None, 4, 4, 32, 32), ([10, 12], [2000, 1500], [7, 0], 5, 5, 40, "none"),
]


def attention_inputs(ops, case, dtype, seed=7):
    nq, nk, gaps, h, hk, d, bias = ATTENTION_CASES[case]
    gen = generator(seed + case)
    seg_q, seg_k = ranges(nq, gaps), ranges(nk, gaps)
    mq, mk = int(seg_q[-1, 1]) + (3 if gaps else 0), int(seg_k[-1, 1]) + (2 if gaps else 0)
    a = dict(q=rand(gen, mq, h, d, dtype=dtype), k=rand(gen, mk, hk, d, dtype=dtype), v=rand(gen, mk, hk, d, dtype=dtype), seg_q=seg_q, seg_k=seg_k)
    go = rand(gen, mq, h, d, dtype=dtype)
    kw = {}
    if bias != "none":
        kw = dict(coords_q=voxel_rows(gen, mq), coords_k=voxel_rows(gen, mk))
        if bias == "slopes":
            kw["slopes"] = 0.05 * 2.0 ** -torch.arange(h, device="cuda").float()
        else:
            kw["bias"], kw["edges"] = rand(gen, bias, h), edges_of(ops, bias)
    return a, kw, go


def reference(a, kw, go, **more):
    names = {"coords_q": "cq", "coords_k": "ck"}
    return attention_ref(**a, **{names.get(n, n): t for n, t in kw.items()}, go=go, **more)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", range(len(ATTENTION_CASES)))
def test_attention_against_64_bits(ops, case, dtype):
    a, kw, go = attention_inputs(ops, case, dtype)
    val, bnd = reference(a, kw, go)
    leaves = [a[n].detach().requires_grad_() for n in "qkv"]
    table = kw["bias"].detach().requires_grad_() if "bias" in kw else None
    call = {**kw, **({} if table is None else {"bias": table})}
    out = ops.segment_attention(*leaves, a["seg_q"].cuda(), a["seg_k"].cuda(), **call)
    grads = torch.autograd.grad(out, leaves + ([] if table is None else [table]), go)
    assert out.dtype == dtype and all(g.dtype == dtype for g in grads[:3])
    what = f"{ATTENTION_CASES[case]} {dtype}"
    for name, got in zip(("out", "dq", "dk", "dv", "dt"), (out.detach(),) + grads):
        assert_within(got, val[name], bnd[name], 1e-30 if name == "dt" else TINY[dtype], f"{name} {what}")
    outside = torch.ones(out.shape[0], dtype=torch.bool)
    for lo, hi in a["seg_q"].tolist():
        outside[lo:hi] = False
    assert (out[outside.cuda()] == 0).all() and (grads[0][outside.cuda()] == 0).all()
    with torch.no_grad():                     # inference: no statistics kept, the same output -- but with a table and 16-bit operands, where
        lean = ops.segment_attention(a["q"], a["k"], a["v"], a["seg_q"].cuda(), a["seg_k"].cuda(), **kw)      # training takes twice the bits
    if table is None or dtype == F32:
        assert torch.equal(lean, out)
    assert_within(lean, val["out"], bnd["out"], TINY[dtype], f"inference {what}")
    again = ops.segment_attention(*leaves, a["seg_q"].cuda(), a["seg_k"].cuda(), **call)
    for one, two in zip(grads, torch.autograd.grad(again, leaves + ([] if table is None else [table]), go)):
        assert torch.equal(one, two)


def test_attention_other_scans_never_reach_a_row(ops):
    """NaN and Inf in another scan's keys and values, and in rows of no scan, stay there (forward and backward)."""
    gen = generator(5)
    seg = ranges([70, 50, 40], [3, 0, 2])
    m = 170
    for dtype in (F32, BF16, F16):
        q, k, v = (rand(gen, m, 4, 32, dtype=dtype) for _ in range(3))
        c, go, slopes = voxel_rows(gen, m), rand(gen, m, 4, 32, dtype=dtype), torch.full((4,), 0.01, device="cuda")
        def both(q, k, v):
            leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
            out = ops.segment_attention(*leaves, seg.cuda(), seg.cuda(), coords_q=c, coords_k=c, slopes=slopes)
            return (out.detach(),) + torch.autograd.grad(out, leaves, go)
        clean = both(q, k, v)
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        for t, bad in ((k2, math.nan), (v2, math.inf), (q2, -math.inf)):
            t[73:123], t[:3], t[123:125], t[165:] = bad, bad, bad, bad          # the second scan and the rows of none
        for x, y in zip(clean, both(q2, k2, v2)):
            assert torch.equal(x[3:73], y[3:73]) and torch.equal(x[125:165], y[125:165])
            assert (y[:3] == 0).all() and (y[165:] == 0).all()


def test_attention_scores_at_the_ends_of_the_range(ops):
    """Scores of the type's lowest value, all equal, far apart; one key; the softmax stays finite and right."""
    for dtype in (F32, BF16, F16):
        big = torch.finfo(dtype).max ** 0.5 / 8
        q = torch.full((20, 2, 32), big, dtype=dtype, device="cuda")
        k = -q[:13].clone()                                        # every score near the lowest value: a plain mean of the values
        v = torch.arange(13, device="cuda").to(dtype)[:, None, None].expand(13, 2, 32).contiguous()
        out = ops.segment_attention(q, k, v, scale=1 / 32)
        assert (out.double() - 6.0).abs().max() <= 6 * torch.finfo(dtype).eps
        k[4] = q[4]                                                # one key takes everything
        assert torch.equal(ops.segment_attention(q, k, v, scale=1 / 32), torch.full_like(out, 4.0))
        lone = ops.segment_attention(q, k[:1], v[5:6], scale=1 / 32)
        assert torch.equal(lone, torch.full_like(out, 5.0))


def test_attention_with_buckets_masked_by_the_lowest_value(ops):
    """Table entries of -inf and of fp32's lowest value: such keys take no part beside others; a row that sees nothing else gives zeros
    (-inf), or the softmax of its scores (the lowest value: the same offset for every key)."""
    gen = generator(16)
    n, edges = 200, (50 * 50,)
    ck = torch.zeros(n, 4, dtype=torch.int32, device="cuda")
    ck[:, 1] = torch.arange(n, device="cuda")                     # keys on a line; queries at 0 and far away from every key
    cq = torch.zeros(6, 4, dtype=torch.int32, device="cuda")
    cq[3:, 1] = 1000
    for dtype in (F32, BF16, F16):
        q, k, v = rand(gen, 6, 2, 32, dtype=dtype), rand(gen, n, 2, 32, dtype=dtype), rand(gen, n, 2, 32, dtype=dtype)
        go = rand(gen, 6, 2, 32, dtype=dtype)
        def both(far):
            leaves = [t.detach().requires_grad_() for t in (q, k, v)] + [torch.tensor([[0.0, 0.5], [far, far]], device="cuda").requires_grad_()]
            out = ops.segment_attention(*leaves[:3], coords_q=cq, coords_k=ck, bias=leaves[3], edges=edges)
            return [out.detach()] + list(torch.autograd.grad(out, leaves, go))
        near = ops.segment_attention(q[:3], k[:50], v[:50], coords_q=cq[:3], coords_k=ck[:50].contiguous(), bias=torch.tensor([[0.0, 0.5]], device="cuda"), edges=())
        plain = both(0.0)
        for far in (-math.inf, torch.finfo(F32).min, -1e9):
            got = both(far)
            assert all(torch.isfinite(t).all() for t in got)
            # (the masked tiles add exact zeros; a table call of another length sums in another order: a few half steps)
            assert (got[0][:3].double() - near.double()).abs().max() <= 8 * torch.finfo(dtype).eps * v.double().abs().max()
            if far == -math.inf:
                assert (got[0][3:] == 0).all() and (got[1][3:] == 0).all()
            else:
                # scores near 2^14 / log2 e / scale have steps of 2^-8 / 0.18 score units' worth: probabilities are off by 2 x 7e-4 at most
                off = (got[0][3:].double() - plain[0][3:].double()).abs().max()
                assert off <= (2 * 7e-4 + 4 * torch.finfo(dtype).eps) * 2 * v.double().abs().max()


def test_attention_buckets_are_exact(ops):
    """A table that spells its bucket, one key per query: every lattice distance up to the last edge and far beyond it."""
    for buckets in (2, 16, 32, 48):
        edges = ops.distance_edges(buckets, 120, 1)
        table = torch.arange(buckets, device="cuda").float()[:, None].contiguous()
        n = 4000
        cq = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
        ck = torch.zeros(n, 4, dtype=torch.int32, device="cuda")
        ck[:, 1] = torch.arange(n, device="cuda") % 500
        ck[:, 2] = torch.arange(n, device="cuda") // 500
        ck[-3:, 1:] = torch.tensor([[32767, -32768, 32767], [-2049, 0, 0], [0, 0, -32768]], device="cuda")
        d2 = ck[:, 1:].long().square().sum(1)
        want = torch.bucketize(d2, torch.tensor(edges, device="cuda"), right=True)
        # the k-th key alone is visible to the k-th query's scan: its weight is 1 whatever the bias, so read the bias from the gradient
        q, k = torch.zeros(n, 1, 32, device="cuda"), torch.zeros(n, 1, 32, device="cuda")
        v = torch.randn(n, 1, 32, generator=generator(3), device="cuda")
        leaf = table.clone().requires_grad_()
        for lo in range(0, n, 500):
            keys = slice(lo, lo + 500)
            out = ops.segment_attention(q[:1], k[keys], v[keys], coords_q=cq, coords_k=ck[keys].contiguous(), bias=leaf, edges=edges)
            p = torch.softmax(want[keys].double(), 0)
            assert torch.allclose(out[0, 0].double(), p @ v[keys, 0].double(), rtol=1e-4, atol=1e-4)      # (a bucket off by one: a factor e)
            go = torch.randn(1, 1, 32, generator=generator(4), device="cuda")
            g, = torch.autograd.grad(out, [leaf], go)
            dp = v[keys, 0].double() @ go[0, 0].double()
            ds = p * (dp - p @ dp)
            assert torch.allclose(g[:, 0].double(), torch.bincount(want[keys], ds, minlength=buckets), rtol=1e-4, atol=1e-5)


def test_attention_keeps_nothing_where_no_gradient_is_asked_for(ops, monkeypatch):
    """Parameters that require gradients, under no_grad: the inference call (no fp32 output, no statistics, one piece), same bits."""
    gen = generator(15)
    q, k, v = (rand(gen, 60, 4, 32, dtype=BF16) for _ in range(3))
    kw = dict(coords_q=voxel_rows(gen, 60), coords_k=voxel_rows(gen, 60), edges=edges_of(ops, 16))
    table = rand(gen, 16, 4)
    want = ops.segment_attention(q, k, v, bias=table, **kw)
    seen = []
    real = ops.call
    monkeypatch.setattr(ops, "call", lambda name, *a, **k: (seen.append(a), real(name, *a, **k))[1])
    with torch.no_grad():
        got = ops.segment_attention(q.clone().requires_grad_(), k, v, bias=table.clone().requires_grad_(), **kw)
    assert torch.equal(got, want) and not got.requires_grad
    assert seen[0][22:25] == (None, 0, None)                     # out_f32, exact, lse


def test_attention_of_a_long_scan_with_the_table_s_gradient(ops):
    """Keys beyond the 64 tiles after which the histogram's words are gathered, every width and type of that kernel, more queries than a
    workgroup takes."""
    for heads, dim, buckets in ((2, 32, 48), (1, 64, 33), (1, 128, 48), (3, 16, 8)):
        for dtype in (F32, BF16, F16):
            gen = generator(heads * dim)
            a = dict(q=rand(gen, 140, heads, dim, dtype=dtype), k=rand(gen, 4300, heads, dim, dtype=dtype), v=rand(gen, 4300, heads, dim, dtype=dtype))
            kw = dict(coords_q=voxel_rows(gen, 140), coords_k=voxel_rows(gen, 4300), bias=rand(gen, buckets, heads), edges=edges_of(ops, buckets))
            go = rand(gen, 140, heads, dim, dtype=dtype)
            val, bnd = reference(a, kw, go)
            leaves = [a[n].requires_grad_() for n in "qkv"] + [kw["bias"].requires_grad_()]
            out = ops.segment_attention(*leaves[:3], **kw)
            for name, got in zip(("out", "dq", "dk", "dv", "dt"), (out.detach(),) + torch.autograd.grad(out, leaves, go)):
                assert_within(got, val[name].detach(), bnd[name].detach(), 1e-30 if name == "dt" else TINY[dtype], f"{name} {heads} x {dim} {dtype}")


def test_table_gradient_s_entries_cancel_over_many_rows(ops):
    """ds of one row sums to zero, so the entries of the table's gradient do: the roundings of 40 000 rows have to fall to both sides.

    A row's own error, with t = sqrt(sum (do out)^2), the size of a partial sum of delta = do . out: 128 additions of delta round by
    2^-24 t / sqrt(3) each (7 of them to the root), some fifty of out's tiles by as much a component (4 of them), the probabilities' pieces
    and the products behind dp by less than one: 12 x 2^-24 t.  Rows are independent, so six times the root of the squares' sum bounds it."""
    rows, dim = 40000, 128
    for dtype in (F16, BF16, F32):
        gen = generator(16)
        q, k, v = (rand(gen, n, 1, dim, dtype=dtype) for n in (rows, 3100, 3100))
        table, go = rand(gen, 32, 1).requires_grad_(), rand(gen, rows, 1, dim, dtype=dtype)
        out = ops.segment_attention(q, k, v, coords_q=voxel_rows(gen, rows), coords_k=voxel_rows(gen, 3100), bias=table, edges=edges_of(ops, 32))
        g, = torch.autograd.grad(out, [table], go)
        root = (out.detach().double() * go.double()).square().sum().sqrt().item()
        assert abs(g.double().sum().item()) <= 6 * 12 * 2.0 ** -24 * root, dtype


def test_attention_layouts(ops):
    """Slices of one fused projection, heads first, one broadcast key row, misaligned storage: the values of contiguous copies."""
    gen = generator(8)
    seg = ranges([90, 61]).cuda()
    for dtype in (F32, BF16):
        qkv = rand(gen, 151, 3, 4, 32, dtype=dtype)
        c, slopes = voxel_rows(gen, 151), torch.full((4,), 0.02, device="cuda")
        kw = dict(coords_q=c, coords_k=c, slopes=slopes)
        want = ops.segment_attention(*(qkv[:, i].contiguous() for i in range(3)), seg, seg, **kw)
        leaf = qkv.clone().requires_grad_()
        out = ops.segment_attention(leaf[:, 0], leaf[:, 1], leaf[:, 2], seg, seg, **kw)
        assert torch.equal(out, want)
        go = rand(gen, 151, 4, 32, dtype=dtype)
        g, = torch.autograd.grad(out, [leaf], go)
        parts = [qkv[:, i].contiguous().requires_grad_() for i in range(3)]
        for i, gp in enumerate(torch.autograd.grad(ops.segment_attention(*parts, seg, seg, **kw), parts, go)):
            assert torch.equal(g[:, i], gp)
        heads_first = [qkv[:, i].transpose(0, 1).contiguous().transpose(0, 1) for i in range(3)]
        assert torch.equal(ops.segment_attention(*heads_first, seg, seg, **kw), want)
        channels_apart = [qkv[:, i].transpose(1, 2).contiguous().transpose(1, 2) for i in range(3)]
        assert torch.equal(ops.segment_attention(*channels_apart, seg, seg, **kw), want)
        odd = torch.zeros(151 * 128 + 1, dtype=dtype, device="cuda")
        odd[1:] = qkv[:, 0].reshape(-1)
        assert torch.equal(ops.segment_attention(odd[1:].view(151, 4, 32), qkv[:, 1], qkv[:, 2], seg, seg, **kw), want)
        # one key head expanded over the query heads: its gradient is the sum of theirs
        k1 = qkv[:, 1, :1].clone().requires_grad_()
        shared = ops.segment_attention(qkv[:, 0], k1, qkv[:, 2, :1], seg, seg, **kw)
        assert torch.equal(ops.segment_attention(qkv[:, 0], k1.expand(151, 4, 32), qkv[:, 2, :1].expand(151, 4, 32), seg, seg, **kw), shared)
        # the gradient of out.sum(): a broadcast gradient
        g1, = torch.autograd.grad(shared.sum(), [k1], retain_graph=True)
        g2, = torch.autograd.grad(shared, [k1], torch.ones_like(shared))
        assert torch.equal(g1, g2)


def test_attention_gradients_against_differences(ops):
    gen = generator(9)
    seg_q, seg_k = ranges([40, 30]).cuda(), ranges([25, 50]).cuda()
    q, k, v = rand(gen, 70, 2, 32), rand(gen, 75, 2, 32), rand(gen, 75, 2, 32)
    kw = dict(coords_q=voxel_rows(gen, 70), coords_k=voxel_rows(gen, 75), edges=edges_of(ops, 16))
    table, go = rand(gen, 16, 2), rand(gen, 70, 2, 32)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    value = lambda ts: (ops.segment_attention(*ts[:3], seg_q, seg_k, bias=ts[3], **kw).double() * go.double()).sum()
    grads = torch.autograd.grad(ops.segment_attention(q, k, v, seg_q, seg_k, bias=table, **kw), leaves, go)
    h = 2.0 ** -7
    for i, g in enumerate(grads):
        step = rand(gen, *g.shape)
        with torch.no_grad():
            moved = lambda s: value([t + (s * h * step if j == i else 0) for j, t in enumerate(leaves)])
            slope = (moved(1.0) - moved(-1.0)) / (2 * h)
        along = (g.double() * step.double()).sum()
        # a central difference: its third-derivative term h^2 / 6 f''' (|f'''| of the order of the cubed steps' scores, bounded here by
        # 60 times the gradient's own size) and the values' fp32 rounding over 2 h
        size = (g.double().abs() * step.double().abs()).sum()
        assert abs(slope - along) <= size * (60 * h * h / 6) + 4 * 2.0 ** -24 * go.double().abs().sum() / (2 * h) * 0.05


def test_group_norm_gradients_against_differences(ops):
    gen = generator(10)
    seg = ranges([50, 21]).cuda()
    x, w, b, dy = rand(gen, 71, 16), 1 + 0.1 * rand(gen, 16), rand(gen, 16), rand(gen, 71, 16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.group_norm(x, 4, w, b, segments=seg, activation="silu"), leaves, dy)
    h = 2.0 ** -7
    for i, g in enumerate(grads):
        step = rand(gen, *g.shape)
        with torch.no_grad():
            moved = lambda s: (ops.group_norm(*(t + (s * h * step if j == i else 0) for j, t in enumerate(leaves[:1])), 4,
                                              *(t + (s * h * step if j + 1 == i else 0) for j, t in enumerate(leaves[1:])), segments=seg,
                                              activation="silu").double() * dy.double()).sum()
            slope = (moved(1.0) - moved(-1.0)) / (2 * h)
        along = (g.double() * step.double()).sum()
        size = (g.double().abs() * step.double().abs()).sum()
        assert abs(slope - along) <= size * (60 * h * h / 6) + 4 * 2.0 ** -24 * dy.double().abs().sum() / (2 * h) * 0.05


def test_refusals_on_the_device(ops):
    q = torch.zeros(8, 2, 32, device="cuda")
    seg = ranges([8])
    with pytest.raises(ValueError, match="is on cpu"):
        ops.segment_attention(q, q, q, seg, seg)
    with pytest.raises(ValueError, match="is on cpu"):
        ops.group_norm(q.view(8, 64), 8, segments=seg)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.segment_attention(q.cpu(), q.cpu(), q.cpu())
    leaf = q.clone().requires_grad_()
    g, = torch.autograd.grad(ops.segment_attention(leaf, q, q).sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# -- segments -----------------------------------------------------------------------------------------------------------------------
def test_batch_segments(ops):
    b = torch.tensor([0] * 5 + [2] * 300 + [3], dtype=torch.int32, device="cuda")
    c = torch.zeros(len(b), 4, dtype=torch.int32, device="cuda")
    c[:, 0] = b
    assert ops.batch_segments(c).tolist() == [[0, 5], [0, 0], [5, 305], [305, 306]]
    assert ops.batch_segments(c, 6).tolist()[4:] == [[0, 0], [0, 0]]
    count = torch.tensor([100], dtype=torch.int32, device="cuda")
    assert ops.batch_segments(c, 4, d_rows=count, replicas=2).tolist() == [[0, 5], [0, 0], [5, 100], [0, 0], [306, 311], [0, 0], [311, 406], [0, 0]]
    assert ops.batch_segments(c, d_rows=count).tolist() == [[0, 5], [0, 0], [5, 100]]
    assert ops.batch_segments(c[:0]).tolist() == [[0, 0]]
    with pytest.raises(ValueError, match="ascending"):
        ops.batch_segments(c.flip(0).contiguous())
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.batch_segments(c.flip(0).contiguous(), 4, status=status)
    assert int(status) == ops.STATUS_BATCH_ORDER


def test_empty_ranges_may_name_any_row(ops):
    """A batch without rows is [0, 0] wherever it stands (batch_segments): no other scan's rows change."""
    gen = generator(14)
    x = rand(gen, 300, 32)
    plain = ranges([5, 200, 95]).cuda()
    holes = torch.tensor([[0, 5], [0, 0], [5, 205], [299, 299], [205, 300], [0, 0]], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.group_norm(x, 8, segments=holes), ops.group_norm(x, 8, segments=plain))
    q = rand(gen, 300, 4, 32)
    assert torch.equal(ops.segment_attention(q, q, q, holes, holes), ops.segment_attention(q, q, q, plain, plain))


def test_ranges_beyond_the_rows_touch_nothing_else(ops):
    """Ranges that leave the row matrix are cut to it (their rows stay inside, no access outside): the documented call has none."""
    gen = generator(11)
    x = rand(gen, 100, 32)
    bad = torch.tensor([[0, 60], [60, 4000], [-5, -1], [2**31 - 1, 2**31 - 1]], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.group_norm(x, 8, segments=bad), ops.group_norm(x, 8, segments=ranges([60, 40, 0, 0]).cuda()))


# -- streams, graphs ----------------------------------------------------------------------------------------------------------------
def _steps(ops, gen):
    """A run of the operators as the attention block uses them: norm -> q, k, v -> attention -> gradients."""
    seg = ranges([150, 90]).cuda()
    x, w, b, table = rand(gen, 240, 128), 1 + 0.1 * rand(gen, 128), 0.1 * rand(gen, 128), rand(gen, 16, 4)
    proj, c, go = 0.1 * rand(gen, 128, 384), voxel_rows(gen, 240), rand(gen, 240, 4, 32)
    edges = edges_of(ops, 16)
    def step(x):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, table)]
        y = ops.group_norm(leaves[0], 16, leaves[1], leaves[2], segments=seg, activation="silu")
        q, k, v = (y @ proj).view(240, 3, 4, 32).unbind(1)
        out = ops.segment_attention(q, k, v, seg, seg, coords_q=c, coords_k=c, bias=leaves[3], edges=edges)
        return (out.detach(),) + torch.autograd.grad(out, leaves, go)
    return x, step


def test_run_of_the_operators_captured_twice_and_replayed(ops):
    gen = generator(12)
    x, step = _steps(ops, gen)
    other = rand(gen, 240, 128)
    want = [t.clone() for t in step(x)]
    want_other = [t.clone() for t in step(other)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    static = x.clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(static))
        graphs.append(g)
    for round_ in range(3):
        for src, ref in ((x, want), (other, want_other)):
            static.copy_(src)
            for g, out in zip(graphs, outs):
                g.replay()
                torch.cuda.synchronize()
                for a, r in zip(out, ref):
                    assert torch.equal(a, r), f"replay {round_}"
            for a, r in zip(step(src), ref):                      # eager work between the replays
                assert torch.equal(a, r)


def test_operators_on_two_streams_at_once(ops):
    gen = generator(13)
    x, step = _steps(ops, gen)
    want = [t.clone() for t in step(x)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step(x))
    torch.cuda.synchronize()
    for res in got:
        for a, r in zip(res, want):
            assert torch.equal(a, r)
