"""Host logic around the scan-wise operators: a library of other sources, limits of a launch, checkpoints, known batches (no GPU)."""
import pytest
import torch


def test_a_library_of_other_sources_is_named_as_such(monkeypatch):
    """A library without an entry point that this package calls (built before it existed) is a version mismatch, not an AttributeError."""
    from lidiff_amd import _lib
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setitem(_lib.SIGNATURES, "lidiff_of_a_later_version", (_lib._i32, []))
    with pytest.raises(RuntimeError, match="version mismatch.*lidiff_of_a_later_version"):
        _lib.load()
    monkeypatch.undo()
    assert _lib.load().lidiff_abi_version() == _lib.ABI_VERSION


def test_a_checkpoint_s_attention_block_is_loaded(tmp_path):
    """The refiner's and the denoiser's attention blocks come back from their checkpoints whatever the other one's hyper-parameters say."""
    from lidiff_amd.diffusion import DiffusionPoints, RefineDiffusion
    from lidiff_amd.pipeline import DiffCompletion
    torch.manual_seed(0)
    paths = {}
    for name, model in (("diff", DiffusionPoints({"model": {"attention_heads": 8}}, device="cpu")), ("plain_diff", DiffusionPoints(device="cpu")),
                        ("refine", RefineDiffusion({"model": {"attention_heads": 4}}, device="cpu")), ("plain_refine", RefineDiffusion(device="cpu"))):
        for key, p in model.named_parameters():
            if ".attention." in key:
                torch.nn.init.normal_(p)
        paths[name] = tmp_path / f"{name}.ckpt"
        torch.save({"state_dict": model.state_dict(), "hyper_parameters": model.hparams}, paths[name])
    for diff in (None, "diff", "plain_diff"):
        for refine in (None, "refine", "plain_refine"):
            pipe = DiffCompletion(diff and paths[diff], refine and paths[refine], device="cpu")
            mine = pipe.state_dict()
            for name in (diff, refine):
                for key, t in (torch.load(paths[name])["state_dict"] if name else {}).items():
                    if ".attention." in key:
                        assert torch.equal(mine[key], t), (name, key)
            assert (pipe.model.attention is not None) == (diff == "diff") and (pipe.model_refine.attention is not None) == (refine == "refine")
    # without a checkpoint, or with one that holds no block, the configuration decides
    assert DiffCompletion(None, None, hparams={"model": {"refine_attention_heads": 4}}, device="cpu").model_refine.attention.num_heads == 4
    # a checkpoint without hyper-parameters
    torch.save({"state_dict": torch.load(paths["diff"])["state_dict"]}, tmp_path / "bare.ckpt")
    assert DiffCompletion(tmp_path / "bare.ckpt", device="cpu").model.attention.num_heads == 8
