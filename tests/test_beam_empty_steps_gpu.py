"""Steps without sequences, laid out on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("width", [0, 3])
def test_a_step_of_no_sequence(width):
    """Its offsets are a zero, and as many pages are taken behind it as before it."""
    from inferloop_b200.csrc import ops
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    none, cu, positions, refused, out = i32([]), i32([-7]), i32([-7, -7]), i32([0]), i32([-7])
    pages = [ops.StepPages(torch.zeros((0, width), dtype=torch.int32, device=DEV), i32([3, 4, 5]), i32([2]), 16, 1, out),
             ops.StepPages(torch.zeros((0, width), dtype=torch.int32, device=DEV), i32([]), i32([0]), 32, 4)]
    slot_map = torch.full((2,), -7, dtype=torch.int64, device=DEV)
    ops.step_build(none, none, none, positions, positions.clone(), cu, pages, refused, slot_map=slot_map)
    assert cu.tolist() == [0] and out.tolist() == [2] and pages[1].used.tolist() == [0] and refused.tolist() == [0]
    assert positions.tolist() == [-7, -7] and slot_map.tolist() == [-7, -7]
    pages[0].used.fill_(9)                                   # (more than there are)
    ops.step_build(none, none, none, positions, positions.clone(), cu.fill_(-7), pages, refused)
    assert refused.tolist() == [2] and cu.tolist() == [-7] and out.tolist() == [2]
