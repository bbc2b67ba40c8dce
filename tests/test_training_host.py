"""The Python layer of the training operators, without a GPU."""
import pytest


@pytest.fixture
def training():
    import __graft_entry__
    __graft_entry__.build()
    from aethelstream_b200 import training
    return training


def test_workspace_sizes_are_kept_per_device(training, monkeypatch):
    """Two devices with different numbers of SMs, in turn: each gets its own size."""
    current, asked = [0], []

    class Library:
        @staticmethod
        def aeth_cut_ce_workspace(n, d, vocab, backward, size):
            asked.append((n, d, vocab, backward))
            size._obj.value = (7, 148)[current[0]] * n
            return 0

    monkeypatch.setattr(training, "_lib", Library)
    training._workspace_bytes.cache_clear()
    try:
        for dev, want in ((0, 70), (1, 1480), (0, 70), (1, 1480)):
            current[0] = dev
            assert training._workspace_bytes("aeth_cut_ce_workspace", dev, 10, 64, 100, 0) == want
        assert asked == [(10, 64, 100, 0)] * 2
    finally:
        training._workspace_bytes.cache_clear()


def test_scales_without_dimensions_are_refused(training):
    """One row of one block: as many scales as are due, but not in the checkpoint's shape."""
    import torch
    ck = training.ActivationCheckpoint(torch.zeros(1, 64, dtype=torch.int8), torch.ones(()), torch.bfloat16)
    with pytest.raises(ValueError, match="ActivationCheckpoint"):
        training._ckpt_args("checkpoint_decode", ck, -1)
