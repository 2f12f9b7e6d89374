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


def test_more_segments_than_a_launch_holds_are_refused():
    """A launch has at most 2^32 threads in a row: more segments x heads (groups, channels) are refused before anything is queued."""
    import ctypes
    from lidiff_amd import _lib
    lib = _lib.load()
    P = lambda i=1: ctypes.c_void_p(4096 * i)                       # (never read: the checks come first)
    word = lambda: lib.lidiff_last_error().decode()
    for segments, c, groups in ((1 << 20, 256, 64), (1 << 20, 1024, 1), (1 << 19, 128, 128)):
        assert lib.lidiff_group_norm(P(), 8, c, groups, 0, P(2), segments, None, None, 1e-5, 0, P(3), P(4), P(5), None) == 1 and "segments x" in word()
        assert lib.lidiff_group_norm_bwd(P(), P(), 8, c, groups, 0, P(2), segments, None, None, P(4), 0, P(3), None, None, P(5), None) == 1 and "segments x" in word()
    strides = (ctypes.c_int64 * 8)(*[512, 32] * 4)
    for segments, heads in ((1 << 20, 8), (1 << 18, 32), (1 << 13, 1024)):
        assert lib.lidiff_segment_attention(P(), P(), P(), strides, None, None, P(2), P(3), segments, 8, 8, heads, heads, 32, 1, 0.2, 0, None, None, None, 0, P(4),
                                            None, 0, None, P(5), None) == 1 and "segments x heads" in word()
        assert lib.lidiff_segment_attention_bwd(P(), P(), P(), P(), strides, None, None, P(2), P(3), segments, 8, 8, heads, heads, 32, 1, 0.2, 0, None, None, None, 0,
                                                P(4), P(5), P(6), P(7), P(8), None, P(9), None) == 1 and "segments x heads" in word()
