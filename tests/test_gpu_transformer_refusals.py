"""GPU: calls of the encoder-layer operators that have no right answer and must say so."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("H,Hk", [(0, 2), (2, 0)])
@pytest.mark.parametrize("train", [False, True])
def test_norm_and_rotation_of_one_side_without_heads(H, Hk, train):
    from asr_amd.Models.transformer_ops import qk_norm_rope
    q, k, w = (torch.ones(s, device=DEV).requires_grad_(train) for s in ((1, 3, H, 8), (1, 3, Hk, 8), (8,)))
    with pytest.raises(RuntimeError, match="do not match"):
        qk_norm_rope(q, k, w, w)


def test_norm_and_rotation_of_nothing():
    from asr_amd.Models.transformer_ops import qk_norm_rope
    for shape in ((1, 3, 0, 8), (0, 3, 2, 8), (1, 0, 2, 8)):
        q, k = (torch.ones(shape, device=DEV).requires_grad_() for _ in range(2))
        w = torch.ones(8, device=DEV).requires_grad_()
        y = qk_norm_rope(q, k, w, w)
        assert all(o.shape == q.shape for o in y)
        assert not torch.autograd.grad(y, w, [torch.ones_like(o) for o in y])[0].any()
