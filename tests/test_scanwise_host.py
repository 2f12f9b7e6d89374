"""Host logic of the scan-wise operators: refusals, the buckets' look-up table, the library's own argument checks (no GPU)."""
import ctypes
import math
import random

import pytest
import torch


@pytest.fixture(scope="module")
def ops():
    from lidiff_amd import ops
    return ops


def test_bucket_cells_name_every_distance_s_bucket(ops):
    """The kernels' rule (cell of the fp32 squared distance, one comparison) against a search, on lattice distances, around every edge and at
    the ends of the range."""
    rng = random.Random(0)
    for edges in (ops.distance_edges(32, 100, 16), ops.distance_edges(48, 120, 8), ops.distance_edges(2, 100, 1), ops.distance_edges(3, 50, 0.5), (), (1,),
                  (1, 2, 3, 4, 5, 9, 1 << 22)):
        cells = ops.bucket_cells(edges)
        d2 = sorted({0, 1, 2, 3, 3 * 65535 ** 2} | {max(0, e + o) for e in edges for o in (-1, 0, 1)} | {rng.randrange(1 << 24) for _ in range(400)})
        f = torch.tensor(d2, dtype=torch.float64).float()
        at = ((f.view(torch.int32) >> 18) - ((127 << 5) - 1)).clamp(0, cells.shape[0] - 1)
        got = (cells[at] & 255) + ((f.view(torch.int32) & ((1 << 18) - 1)) >= (cells[at] >> 8)).int()
        assert got.tolist() == [sum(e <= v for e in edges) for v in d2]
        assert int((cells & 255).max()) <= len(edges)


def test_edges_are_refused(ops):
    for bad in ((0,), (4, 4), (9, 4), (1.5,), ((1 << 22) + 1,), (10000, 10001)):
        with pytest.raises(ValueError):
            ops.bucket_cells(bad)
    for args in ((0, 10), (49, 100), (8, 3), (8, 100, 0.0), (8, 100, -1.0), (32, 1e6, 16)):
        with pytest.raises(ValueError):
            ops.distance_edges(*args)
    assert ops.distance_edges(1, 0) == ()


def test_group_norm_refusals(ops):
    x = torch.zeros(10, 32)
    seg = torch.tensor([[0, 10]], dtype=torch.int32)
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(x=torch.zeros(4, 30)), dict(x=torch.zeros(4, 2048)), dict(num_groups=5), dict(num_groups=0),
                dict(activation="gelu"), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(weight=torch.ones(31)), dict(bias=torch.ones(32, 1)),
                dict(weight=torch.ones(32, dtype=torch.int32)), dict(segments=seg.long()), dict(segments=seg[0]), dict(segments=seg[:0])):
        with pytest.raises(ValueError):
            ops.group_norm(**{"x": x, "num_groups": 8, **bad})
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.group_norm(x, 8, segments=seg)


def test_attention_refusals(ops):
    t = torch.zeros(10, 4, 32)
    c, seg = torch.zeros(10, 4, dtype=torch.int32), torch.tensor([[0, 10]], dtype=torch.int32)
    ok = dict(q=t, k=t, v=t)
    slopes, table = torch.ones(4), torch.zeros(3, 4)
    for bad in (dict(q=t[0]), dict(k=t[:5]), dict(k=t[:, :, :16], v=t[:, :, :16]), dict(q=t.bfloat16()), dict(q=t.double(), k=t.double(), v=t.double()),
                dict(k=t[:, :3], v=t[:, :3]), dict(k=t[:, :0], v=t[:, :0]), dict(zip("qkv", [torch.zeros(10, 4, 36)] * 3)), dict(zip("qkv", [torch.zeros(10, 4, 136)] * 3)),
                dict(seg_q=seg), dict(seg_q=seg, seg_k=torch.cat([seg, seg])), dict(seg_q=seg.long(), seg_k=seg.long()),
                dict(slopes=slopes), dict(slopes=slopes[:3], coords_q=c, coords_k=c), dict(slopes=slopes.requires_grad_(), coords_q=c, coords_k=c),
                dict(bias=table, coords_q=c, coords_k=c), dict(edges=(1, 4)), dict(bias=table, edges=(1,), coords_q=c, coords_k=c),
                dict(bias=table, edges=(1, 4), coords_q=c.long(), coords_k=c), dict(bias=table, edges=(1, 4), coords_q=c[:5], coords_k=c),
                dict(bias=torch.zeros(49, 4), edges=tuple(range(1, 49)), coords_q=c, coords_k=c), dict(bias=table.t(), edges=(1, 4), coords_q=c, coords_k=c),
                dict(bias=table, edges=(1, 4), slopes=torch.ones(4), coords_q=c, coords_k=c), dict(scale=math.inf), dict(scale=math.nan), dict(scale=0.0), dict(scale=-1.0)):
        with pytest.raises(ValueError):
            ops.segment_attention(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.segment_attention(t, t, t, seg, seg)


def test_batch_segments_refusals(ops):
    c = torch.zeros(10, 4, dtype=torch.int32)
    for args in ((c.long(),), (c[:, :3],), (c, 0), (c, 1, None, 0), (c, 1, torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.batch_segments(*args)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.batch_segments(c)


def test_library_refuses_before_it_launches():
    """Every call is rejected by the library's own checks: none gets as far as a launch."""
    from lidiff_amd import _lib
    lib = _lib.load()
    P = lambda i=1: ctypes.c_void_p(4096 * i)                       # (never read: the checks come first)
    good = dict(rows=8, c=32, groups=8, dtype=0, seg=P(), nseg=1, act=0, x=P(), y=P(2))
    def norm(**kw):
        a = {**good, **kw}
        rc = lib.lidiff_group_norm(a["x"], a["rows"], a["c"], a["groups"], a["dtype"], a["seg"], a["nseg"], None, None, 1e-5, a["act"], a["y"], P(3), P(4), None)
        return rc, lib.lidiff_last_error().decode()
    for kw, word in ((dict(x=None), "null"), (dict(rows=0), "rows"), (dict(c=30), "multiple of 4"), (dict(c=2048), "multiple of 4"), (dict(groups=5), "divide"),
                     (dict(dtype=3), "dtype"), (dict(nseg=0), "segments"), (dict(nseg=2, seg=None), "one"), (dict(act=3), "activation"),
                     (dict(x=ctypes.c_void_p(4100)), "misaligned"), (dict(rows=2 ** 31), "rows"),
                     (dict(rows=2 ** 30, c=512), "channels")):
        rc, msg = norm(**kw)
        assert rc == 1 and word in msg, (kw, msg)
    base = dict(q=P(), k=P(2), v=P(3), strides=[128, 32] * 3, cq=P(4), ck=P(5), sq=P(6), sk=P(7), nseg=1, mq=8, mk=8, h=4, hk=4, d=32, dtype=0, mode=0, scale=0.1, slopes=None,
                table=None, cells=None, buckets=0, out=P(8))
    def attend(**kw):
        a = {**base, **kw}
        rc = lib.lidiff_segment_attention(a["q"], a["k"], a["v"], (ctypes.c_int64 * 6)(*a["strides"]), a["cq"], a["ck"], a["sq"], a["sk"], a["nseg"], a["mq"], a["mk"],
                                          a["h"], a["hk"], a["d"], a["dtype"], a["scale"], a["mode"], a["slopes"], a["table"], a["cells"], a["buckets"], a["out"], None, 0,
                                          None, None, None)
        return rc, lib.lidiff_last_error().decode()
    for kw, word in ((dict(q=None), "null"), (dict(k=None), "null"), (dict(sq=None), "together"), (dict(nseg=0), "segments"), (dict(mq=0), "rows"), (dict(mk=-1), "rows"),
                     (dict(mq=2 ** 31), "rows"), (dict(mq=2 ** 28), "2^26"), (dict(mk=2 ** 28), "2^26"), (dict(hk=3), "divide"), (dict(d=36), "head dimension"), (dict(d=256), "head dimension"), (dict(dtype=7), "dtype"),
                     (dict(mode=3), "bias"), (dict(mode=1), "null"), (dict(mode=1, cq=None, slopes=P()), "coordinates"), (dict(mode=2, buckets=49), "buckets"),
                     (dict(mode=2, buckets=8), "null"), (dict(strides=[127, 32] * 3), "16-byte"), (dict(strides=[-128, 32] * 3), "16-byte"), (dict(strides=[1 << 22, 32] * 3), "row stride"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
                     (dict(q=ctypes.c_void_p(4104)), "misaligned"), (dict(mk=5000), "workspace missing")):
        rc, msg = attend(**kw)
        assert rc == 1 and word in msg, (kw, msg)
    assert lib.lidiff_segment_attention_workspace_bytes(8, 5000, 1, 4, 4, 32, 1, 0) > 0
    assert lib.lidiff_segment_attention_workspace_bytes(8, 5000, 1, 4, 3, 32, 1, 0) == 0
    assert lib.lidiff_segment_attention_bwd_workspace_bytes(8, 8, 1, 4, 4, 32, 1, 2, 16, 1) >= 8 * 4 * 4
    rc = lib.lidiff_batch_segments(P(), 2 ** 30, None, 4, 4, P(2), P(3), None)
    assert rc == 1 and "2^31" in lib.lidiff_last_error().decode()
