"""Row ranges of a batch's scans where the number of scans is known: no host read of it, the ranges that the read would give (MI355X)."""
import pytest
import torch

from test_gpu_scanwise_models import small_batch, training_model

pytestmark = pytest.mark.gpu


@pytest.fixture
def asked(monkeypatch):
    """Every call of ops.batch_segments: (number of batches handed in, coordinates, row count, replicas, result)."""
    from lidiff_amd import ops
    seen, real = [], ops.batch_segments
    def record(coords, n_batches=None, d_rows=None, replicas=1, status=None):
        seen.append((n_batches, coords, d_rows, replicas, real(coords, n_batches, d_rows=d_rows, replicas=replicas, status=status)))
        return seen[-1][-1]
    monkeypatch.setattr(ops, "batch_segments", record)
    yield seen
    for n, coords, d_rows, replicas, got in seen:
        want = real(coords, None, d_rows=d_rows)
        assert n is not None and n >= want.shape[0] and (got[:want.shape[0]] == want).all() and (got[want.shape[0]:n] == 0).all()


@pytest.mark.parametrize("scans", [1, 2, 3])
def test_training_knows_its_scans(device, asked, scans):
    model = training_model(device)
    model.training_step(small_batch(scans, 1200), noise=torch.zeros(scans, 1200, 3), t=torch.tensor([500, 100, 900][:scans]), drop=False).backward()
    assert len(asked) >= 2


@pytest.mark.parametrize("scans,resolution", [(1, 0.05), (2, 0.05), (3, 0.05), (2, 0.4), (3, 0.07)])
def test_refinement_knows_its_scans(device, asked, scans, resolution):
    """(The batch column is divided by the resolution: two scans are batches 0 and 20.)"""
    from lidiff_amd.diffusion import RefineDiffusion
    torch.manual_seed(4)
    model = RefineDiffusion({"model": {"attention_heads": 4}, "data": {"resolution": resolution}}, device=device).train()
    full = small_batch(scans, 1200)["pcd_full"].to(device)
    model.training_step({"pcd_noise": full + 0.01 * torch.randn_like(full), "pcd_full": full}).backward()
    assert asked


@pytest.mark.parametrize("scans", [1, 2])
@pytest.mark.parametrize("fused", [True, False])
def test_fields_of_the_pipeline_know_their_scans(device, asked, scans, fused):
    from lidiff_amd.pipeline import DiffCompletion
    pipe = DiffCompletion(denoising_steps=4, device=device, hparams={"model": {"attention_heads": 8}})
    pipe.fused_step = fused
    x = pipe.points_to_tensor(small_batch(scans, 1000)["pcd_full"].to(device)).sparse()
    assert x.segments().shape[0] == (1 if scans == 1 else 21)
    assert len(asked) == 1


def test_farthest_points_where_the_cooperative_launch_is_refused(device, monkeypatch):
    """The warning gives the library's reason, whatever it is; the indices are those of the cooperative launch."""
    from lidiff_amd import _lib, ops
    points = torch.randn(3000, 3, dtype=torch.float64, generator=torch.Generator().manual_seed(5)).to(device)
    want, real = ops.farthest_point_sample(points, 100), ops.call
    class Library:
        def __getattr__(self, name):
            return getattr(lib, name)
        def lidiff_last_error(self):
            return b"lidiff_fps_coop: the runtime refuses the cooperative launch now (a reason of its own)"
    lib = _lib.load()
    monkeypatch.setattr(ops, "call", lambda name, *a, **k: 3 if name == "lidiff_fps_coop" else real(name, *a, **k))
    monkeypatch.setattr(_lib, "load", lambda: Library())
    with pytest.warns(UserWarning, match="a reason of its own.*running lidiff_fps"):
        got = ops.farthest_point_sample(points, 100)
    assert torch.equal(got, want)
