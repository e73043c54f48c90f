"""What the appends take as ``position_offset``: a whole number, or int32 [B] on the device (no GPU)."""

import pytest
import torch

from flash_topk_attn_v2.qk_prep import offsets

CPU = torch.device("cpu")


@pytest.mark.parametrize("x", [torch.tensor([5]), torch.tensor([[5]]), torch.tensor([5.0]), torch.tensor([[5]], dtype=torch.int32),
                               torch.tensor([5], dtype=torch.int16)], ids=str)
@pytest.mark.parametrize("B", [1, 2])
def test_one_element_is_a_number(x, B):
    """As it was before there were offsets of each request."""
    assert offsets("append", x, B, CPU, 64, 8) == (5, None)


def test_one_offset_of_one_request():
    """int32 [1] is the offset of each request of one, or, elsewhere than on the device, a number; of more requests
    it is neither."""
    x = torch.tensor([5], dtype=torch.int32)
    number, each = offsets("append", x, 1, CPU, 64, 8)
    assert number == 0 and each.tolist() == [5]
    assert offsets("append", x, 1, torch.device("meta"), 64, 8) == (5, None)
    with pytest.raises(ValueError, match="whole number"):
        offsets("append", x, 3, CPU, 64, 8)


@pytest.mark.parametrize("x", [torch.tensor([0.5]), torch.tensor([float("nan")]), torch.tensor([1 << 31]), torch.tensor([3, 4]),
                               torch.tensor([3.0, 4.0]), torch.zeros(0, dtype=torch.int32), torch.tensor([[3, 4]], dtype=torch.int32)], ids=str)
def test_what_is_neither_is_refused(x):
    with pytest.raises(ValueError):
        offsets("append", x, 2, CPU, 64, 8)


def test_offsets_of_another_device_are_refused():
    with pytest.raises(ValueError, match="expected meta"):
        offsets("append", torch.tensor([3, 4], dtype=torch.int32), 2, torch.device("meta"), 64, 8)
