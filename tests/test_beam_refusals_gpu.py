"""Calls of the beam search operators whose result would depend on the order of writes, or would be none: refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from inferloop_b200.csrc import ops
    return ops


def z(*shape, dt=torch.int32):
    return torch.zeros(*shape, dtype=dt, device=DEV)


def test_one_block_table_for_two_groups(ops):
    """A table follows its beams once a group: twice would take it to the parents' parents."""
    caches = [z(2, 9, 2, 16, 64, dt=torch.float32) for _ in range(2)]
    state = ops.BeamState([([c], 16, 1) for c in caches])
    both = z(16, 4)
    parents, kv_len = z(2, 4), z(8)
    for tables in ((both[:8], both[:8]), (both[:8], both[7:15])):
        with pytest.raises(ops.KernelError, match="share memory"):
            ops.beam_reorder(state, parents, kv_len, tables)
    ops.beam_reorder(state, parents, kv_len, (both[8:], both[:8]))
    a = z(4)
    page = lambda table, used, out=None: ops.StepPages(table, z(5), used, 16, 1, out)  # noqa: E731
    for tables in ((both[:4], both[:4]), (both[:4], both[3:7])):
        with pytest.raises(ops.KernelError, match="share memory"):
            ops.step_build(a, a, a, z(4), z(4), z(5), [page(t, z(1)) for t in tables], z(1))
    ops.step_build(a, a, a, z(4), z(4), z(5), [page(t, z(1)) for t in (both[4:8], both[:4])], z(1))


def test_one_count_of_pages_for_two_groups(ops):
    """Two groups that take pages by one counter would take the same ones."""
    a, one, two = z(4), z(1), z(1)
    page = lambda used, out=None: ops.StepPages(z(4, 3), z(5), used, 16, 1, out)  # noqa: E731
    for pages in ([page(one), page(one)], [page(one, two), page(z(1), two)], [page(one), page(z(1)), page(one, two)], [page(one, two), page(two)]):
        with pytest.raises(ops.KernelError, match="in one place"):
            ops.step_build(a, a, a, z(4), z(4), z(5), pages, z(1))
    ops.step_build(a, a, a, z(4), z(4), z(5), [page(one, two), page(one, z(1))], z(1))         # (the same number read twice)


@pytest.mark.parametrize("last,penalty,served", [(2, 100.0, True), (2, -100.0, True), (2, 101.0, False), (16, 25.5, False), (16, -25.5, False), (4, float("nan"), False),
                                                 (4, float("inf"), False), (1, 1e30, True), (1, float("nan"), False), (1, 1e300, False), (3, 1e300, False)])
def test_length_penalties(ops, last, penalty, served):
    """A power that 32 bits do not hold made all scores zero, infinite or NaN."""
    track = ops.BeamTrack.make(1, 2, last, DEV)
    args = (z(1, 2), torch.tensor([[1, 2]], dtype=torch.int32, device=DEV), torch.tensor([[-1.0, -1.5]], device=DEV), None, track, last - 1, last, penalty)
    if not served:
        with pytest.raises(ops.KernelError, match="power"):
            ops.beam_keep(*args)
        return
    ops.beam_keep(*args)
    want = torch.tensor([-1.0, -1.5], dtype=torch.float64) / float(last) ** penalty
    assert bool(((track.done_scores[0].cpu().double() - want).abs() <= 2.0 ** -21 * want.abs()).all())


def test_heads_of_a_page_of_two_gigabytes(ops):
    """A copy counts the bytes of a page's head in 32 bits: just below 2^31 it moves them, at 2^31 the storage is refused."""
    rows = 1 << 16
    with pytest.raises(ops.KernelError, match="too long"):
        ops.BeamState([([torch.empty((2, 1, rows, 1 << 15), dtype=torch.uint8, device=DEV)], rows, 1)])
    x = torch.zeros((2, 1, rows, (1 << 15) - 16), dtype=torch.uint8, device=DEV)
    x[0, 0, :, -1] = torch.arange(rows, device=DEV).to(torch.uint8)
    table = torch.tensor([[0], [1]], dtype=torch.int32, device=DEV)
    state = ops.BeamState([([x], rows, 1)])
    ops.beam_reorder(state, z(1, 2), torch.full((2,), rows - 1, dtype=torch.int32, device=DEV), [table])
    assert torch.equal(x[1, 0, :-1], x[0, 0, :-1]) and int(x[1, 0, -1].sum()) == 0
