"""CPU: what the native module of the encoder-layer operators refuses before it looks for a GPU."""
import pytest
import torch


def _native():
    from asr_amd import _lib
    return _lib.native()


@pytest.mark.parametrize("H,Hk", [(0, 2), (2, 0)])
def test_norm_and_rotation_of_one_side_without_heads(H, Hk):
    """The other side must not come back as memory that nobody wrote."""
    q, k, w = torch.ones(1, 3, H, 8), torch.ones(1, 3, Hk, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="both or none"):
        _native().rope_fwd(q, k, w, w, None, 8, 1e4, 1e-6)
    with pytest.raises(RuntimeError, match="both or none"):
        _native().rope_bwd(q, k, w, w, None, 8, 1e4, 1e-6, q, k)


@pytest.mark.parametrize("shape", [(1, 3, 0, 8), (0, 3, 2, 8), (1, 0, 2, 8)])
def test_norm_and_rotation_of_nothing(shape):
    q, w = torch.ones(shape), torch.ones(8)
    for out in _native().rope_fwd(q, q, w, w, None, 8, 1e4, 1e-6):
        assert out.shape == q.shape
    dq, dk, dwq, dwk = _native().rope_bwd(q, q, w, w, None, 8, 1e4, 1e-6, q, q)
    assert dq.shape == dk.shape == q.shape and not dwq.any() and not dwk.any()
