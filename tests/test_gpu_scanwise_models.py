"""The scan-wise operators in the framework's modules and networks: ME.MinkowskiGroupNorm, ME.MinkowskiAttention, the UNets' attention_heads."""
import copy

import numpy as np
import pytest
import torch

from conftest import small_scene
from scanwise_ref import plain_group_norm, plain_segment_attention

pytestmark = pytest.mark.gpu


def scans_tensor(device, sizes, channels, seed, stride=1, extent=30):
    """A sparse tensor of several scans with random features on the map of `stride`."""
    import lidiff_amd.MinkowskiEngine as ME
    rng = np.random.default_rng(seed)
    c = np.concatenate([np.concatenate([np.full((n, 1), b), rng.integers(-extent, extent, (n, 3))], 1) for b, n in enumerate(sizes)]).astype(np.int32)
    sp = ME.SparseTensor(torch.zeros(len(c), 4, device=device), torch.from_numpy(c).to(device), device=device)
    ts = 1
    while ts < stride:
        ts = sp.coordinate_manager.stride(ts, 2)
    m = sp.coordinate_manager.maps[ts].coords.shape[0]
    gen = torch.Generator(device=device).manual_seed(seed)
    return ME.SparseTensor(torch.randn(m, channels, generator=gen, device=device), tensor_stride=ts, coordinate_manager=sp.coordinate_manager)


def wake(block, seed=0):
    """Random values where a new block starts at zero."""
    gen = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in [block.proj.weight, block.proj.bias, block.feed.weight, block.feed.bias, block.distance_bias]:
            p.copy_(0.3 * torch.randn(p.shape, generator=gen))
        for n in (block.norm, block.norm_context, block.norm_feed):
            if n is not None:
                n.weight.copy_(1 + 0.1 * torch.randn(n.weight.shape, generator=gen))
                n.bias.copy_(0.1 * torch.randn(n.bias.shape, generator=gen))


class plain:
    """ops' two operators replaced by their 64-bit forms."""
    def __init__(self, monkeypatch):
        self.mp = monkeypatch

    def __enter__(self):
        from lidiff_amd import ops
        self.ctx = self.mp.context()
        mp = self.ctx.__enter__()
        mp.setattr(ops, "group_norm", plain_group_norm)
        mp.setattr(ops, "segment_attention", plain_segment_attention)

    def __exit__(self, *exc):
        self.ctx.__exit__(*exc)


def close(a, b, rel, what):
    """2-norm of the difference over that of the value: the operators' fp32 roundings (each test of them bounds these) pass through a few
    Linears and sums of up to 10^3 terms: 64 half steps of fp32."""
    off, size = (a.double() - b.double()).norm().item(), b.double().norm().item()
    assert off <= rel * max(size, 1e-30), f"{what}: {off / max(size, 1e-30):.2e}"


REL = 64 * 2.0 ** -24 * 8


def test_segments_of_maps_and_replicas(device):
    x = scans_tensor(device, [500, 1, 300], 8, 1, stride=4)
    seg = x.segments().tolist()
    b = x.C[:, 0].tolist()
    assert len(seg) == 3 and all(set(b[lo:hi]) == {i} for i, (lo, hi) in enumerate(seg)) and seg[-1][1] == len(b)
    assert x.segments() is x.segments()
    twice = x.replicate(2)
    assert twice.segments().tolist() == seg + [[lo + len(b), hi + len(b)] for lo, hi in seg]
    assert x.segments(5).tolist() == seg + [[0, 0], [0, 0]]


@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_group_norm_module(device, act):
    import lidiff_amd.MinkowskiEngine as ME
    x = scans_tensor(device, [400, 7, 300], 48, 2, stride=2)
    mod = ME.MinkowskiGroupNorm(12, 48, activation=act).to(device)
    with torch.no_grad():
        mod.weight.uniform_(0.5, 1.5)
        mod.bias.normal_()
    got = mod(x)
    want = plain_group_norm(x.F, 12, mod.weight, mod.bias, x.segments(), 1e-5, act)
    close(got.F, want, REL, act)
    assert got.tensor_stride == 2 and got.coordinate_manager is x.coordinate_manager
    assert sorted(mod.state_dict()) == ["bias", "weight"]
    with pytest.raises(ValueError):
        ME.MinkowskiGroupNorm(5, 48)
    with pytest.raises(ValueError):
        ME.MinkowskiGroupNorm(4, 48, activation="tanh")


@pytest.mark.parametrize("kv_heads", [4, 1])
@pytest.mark.parametrize("cross", [False, True])
def test_attention_module_and_its_gradients(device, cross, kv_heads, monkeypatch):
    import lidiff_amd.MinkowskiEngine as ME
    x = scans_tensor(device, [900, 5, 700], 64, 3, stride=4)
    part = scans_tensor(device, [300, 250, 1], 48, 4, stride=2)
    torch.manual_seed(0)
    block = ME.MinkowskiAttention(64, 4, context_channels=48 if cross else None, num_kv_heads=kv_heads, unit=4).to(device)
    assert torch.equal(block(x, part if cross else None).F, x.F)                  # a new block is the identity
    wake(block)
    leaf, part_leaf = x.F.clone().requires_grad_(), part.F.clone().requires_grad_()
    go = torch.randn(x.F.shape, generator=torch.Generator(device=device).manual_seed(9), device=device)
    leaves = [leaf] + ([part_leaf] if cross else []) + list(block.parameters())
    def both():
        y = block(x._like(leaf), part._like(part_leaf) if cross else None).F
        return (y.detach(),) + torch.autograd.grad(y, leaves, go)
    got = both()
    with plain(monkeypatch):
        want = both()
    names = ["y", "dx"] + (["dcontext"] if cross else []) + [n for n, _ in block.named_parameters()]
    for n, a, b in zip(names, got, want):
        close(a, b, REL * (8 if n == "distance_bias" else 1), n)                    # (a table entry: sums over rows that cancel)


def test_attention_module_of_a_guidance_pair(device):
    """Two replicas with a context each, as one stacked pass, against the two passes."""
    import lidiff_amd.MinkowskiEngine as ME
    x = scans_tensor(device, [1200], 64, 5, stride=4)
    parts = scans_tensor(device, [400], 64, 6, stride=2), scans_tensor(device, [1], 64, 7)
    block = ME.MinkowskiAttention(64, 2, context_channels=64, unit=4).to(device)
    wake(block)
    with torch.no_grad():
        pair = block(x.replicate(2), parts).F
        for i, p in enumerate(parts):
            close(pair[i * x.F.shape[0]:(i + 1) * x.F.shape[0]], block(x, p).F, REL, i)
        with pytest.raises(ValueError):
            block(x, parts)
        with pytest.raises(ValueError):
            block(x)


def small_batch(b, n):
    pts = [small_scene(seed=20 + i, n=n)[0] for i in range(b)]
    full = torch.from_numpy(np.stack(pts))
    return {"pcd_full": full, "pcd_part": full[:, :n // 10].contiguous()}


def training_model(device, precision="32"):
    from lidiff_amd.diffusion import DiffusionPoints
    torch.manual_seed(1)
    model = DiffusionPoints({"model": {"attention_heads": 8}}, device=device, precision=precision)
    wake(model.model.attention)
    return model.train()


def test_training_step_with_attention(device, monkeypatch):
    """Loss and every parameter gradient of a training step of two scans, against the same step with the operators' 64-bit forms."""
    model = training_model(device)
    batch = small_batch(2, 1500)
    draws = dict(noise=torch.randn(batch["pcd_full"].shape, generator=torch.Generator().manual_seed(3)), t=torch.tensor([700, 200]), drop=False)
    start = copy.deepcopy(model.state_dict())
    def step():
        model.load_state_dict(start)
        loss = model.training_step(batch, **draws)
        return [loss.detach()] + list(torch.autograd.grad(loss, list(model.parameters())))
    got = step()
    with plain(monkeypatch):
        want = step()
        # what a rounding behind the block does to the rest of the network (ReLUs and BatchNorms turn last bits into directions): the
        # operators' own fp32 errors are at most some 16 half steps of their outputs (test_gpu_scanwise.py), so the same step with the
        # block's output moved by as much is the scale that the others' gradients are held to
        block = model.model.attention
        hook = block.register_forward_hook(lambda m, i, y: y._like(y.F * (1 + 16 * 2.0 ** -24 * torch.empty_like(y.F).uniform_(-1, 1, generator=gen))))
        gen = torch.Generator(device=device).manual_seed(0)
        moved = step()
        hook.remove()
    names = ["loss"] + [n for n, _ in model.named_parameters()]
    assert any("attention.distance_bias" in n for n in names)
    for n, a, b, c in zip(names, got, want, moved):
        assert torch.isfinite(a).all(), n
        if n == "loss":
            close(a, b, 1e-5, n)
        elif b.norm() > 1e-6:
            off, scale = ((t.double() - b.double()).norm() / b.double().norm() for t in (a, c))
            assert off <= 4 * scale + REL, (n, off.item(), scale.item())


def test_training_step_in_bf16_runs_the_attention_in_bf16(device, monkeypatch):
    from lidiff_amd import ops
    model = training_model(device, "bf16")
    seen = []
    real = ops.segment_attention
    monkeypatch.setattr(ops, "segment_attention", lambda q, *a, **k: (seen.append(q.dtype), real(q, *a, **k))[1])
    loss = model.training_step(small_batch(2, 1200), noise=torch.zeros(2, 1200, 3), t=torch.tensor([500, 100]), drop=False)
    loss.backward()
    assert seen == [torch.bfloat16]
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.model.attention.parameters())
    assert model.model.attention.distance_bias.grad.abs().sum() > 0


def test_networks_without_attention_keep_their_state_dict_and_values(device):
    from lidiff_amd import minkunet
    torch.manual_seed(2)
    plain_net = minkunet.MinkUNet(in_channels=3, out_channels=18).to(device).eval()
    torch.manual_seed(2)
    with_attention = minkunet.MinkUNet(in_channels=3, out_channels=18, attention_heads=4).to(device).eval()
    extra = set(with_attention.state_dict()) - set(plain_net.state_dict())
    assert extra and all(k.startswith("attention.") for k in extra) and not set(plain_net.state_dict()) - set(with_attention.state_dict())
    with_attention.load_state_dict(plain_net.state_dict(), strict=False)
    import lidiff_amd.MinkowskiEngine as ME
    scan = torch.from_numpy(small_scene(seed=3, n=1500)[0]).to(device)
    def field():
        c = torch.cat([torch.zeros(len(scan), 1, device=device), (scan / 0.05).round()], 1)
        return ME.TensorField(features=scan, coordinates=c, device=device)
    with torch.no_grad():
        assert torch.equal(plain_net(field()), with_attention(field()))           # (a new block is the identity)


@pytest.fixture(scope="module")
def denoiser(device):
    """The seeded networks of the other tests, the UNet with an attention block."""
    from conftest import build_seeded_models
    from lidiff_amd import minkunet
    enc, unet, refine = build_seeded_models(42)
    with_attention = minkunet.MinkUNetDiff(in_channels=3, attention_heads=8)
    with_attention.load_state_dict(unet.state_dict(), strict=False)
    wake(with_attention.attention)
    return enc.to(device).eval(), with_attention.to(device).eval(), refine.to(device).eval()


def pipeline(device, nets, steps, **flags):
    from lidiff_amd.pipeline import DiffCompletion
    pipe = DiffCompletion(denoising_steps=steps, cond_weight=6.0, device=device)
    pipe.partial_enc, pipe.model, pipe.model_refine = nets
    for k, v in flags.items():
        setattr(pipe, k, v)
    pipe.new_scheduler()
    return pipe


def test_denoising_loop_with_attention_without_host_reads(device, denoiser, fps_scan):
    """completion_loop with an attention block: without host reads (maps at their bounds, rows behind the counts; no step voided), and with
    each step's sizes read; run twice without: the same points bit for bit.  The two forms split the keys among workgroups by different
    row counts, so they agree within fp32 summation order, as the two forms of the loop do without attention."""
    import warnings
    steps = 4
    scan = torch.from_numpy(np.tile(fps_scan[:1500], (10, 1))).double()[None].to(device)
    g = torch.Generator().manual_seed(11)
    x0 = (scan.cpu() + 0.6 * torch.randn(scan.shape, generator=g, dtype=torch.float64)).to(device)
    zs = [torch.randn(scan.shape, generator=g, dtype=torch.float64).to(device) for _ in range(steps)]
    def loop(**flags):
        pipe = pipeline(device, denoiser, steps, **flags)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            out = pipe.completion_loop(scan, pipe.points_to_tensor(x0, role="x_t"), pipe.points_to_tensor(scan, role="cond"),
                                       pipe.points_to_tensor(torch.zeros_like(scan), role="uncond"), noises=zs)
        torch.cuda.synchronize()
        return out
    free, again, own = loop(read_free=True), loop(read_free=True), loop(read_free=False)
    assert np.isfinite(free).all() and np.array_equal(free, again)
    assert np.median(np.abs(free - own).max(axis=1)) <= 1e-5


def test_guidance_pair_with_attention_stacked_and_apart(device, denoiser, fps_scan):
    """The guidance pair as one stacked pass (two replicas, a context each) and as two forwards in the reference's op order."""
    scan = torch.from_numpy(np.tile(fps_scan[:1000], (10, 1))).double()[None].to(device)
    outs = []
    for pair in (True, False):
        pipe = pipeline(device, denoiser, 4, read_free=False, pair_cfg=pair)
        noise = torch.randn(scan.shape, generator=torch.Generator().manual_seed(6), dtype=torch.float64).to(device)
        with torch.no_grad():
            e = pipe.classfree_pair(pipe.points_to_tensor(scan + noise), pipe.points_to_tensor(scan), pipe.points_to_tensor(torch.zeros_like(scan)),
                                    torch.tensor([700], device=device))
        outs.append(torch.stack([t.reshape(-1, 3) for t in e]))
    close(outs[0], outs[1], 1e-5, "pair")
