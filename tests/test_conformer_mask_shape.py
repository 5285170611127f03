"""CPU: the Conformer encoder refuses a frame mask that does not belong to its frames before any kernel reads it."""
import pytest
import torch


@pytest.mark.parametrize("attention", ["relative", "rotary", "bucket"])
@pytest.mark.parametrize("bad", ["short", "one row", "dtype", "strides"])
def test_mask_of_other_frames(attention, bad):
    from asr_amd.Models.Transformer_encoder import ConformerEncoder
    m = ConformerEncoder(64, 1, 4, 0.0, attention)
    src, keep = torch.zeros(2, 9, 64), torch.ones(2, 9, dtype=torch.uint8)
    keep = {"short": keep[:, :7].contiguous(), "one row": keep[:1], "dtype": keep.long(), "strides": keep.t().contiguous().t()}[bad]
    with pytest.raises(RuntimeError, match="keep must be"):
        m(src, keep)
