"""The 4-bit cache's geometry and what is refused before any device is asked."""
import pytest
import torch

from inferloop_b200.csrc import ops


def test_shape_and_bytes():
    assert ops.kv4_cache_shape(7, 8, 64, 128) == (7, 8, 4, 2304)
    # 4.5 bits an element of keys and values
    assert 7 * 8 * 4 * 2304 * 8 == 7 * 8 * 64 * 128 * 2 * 4.5


@pytest.mark.parametrize("page,d", [(8, 64), (0, 64), (-16, 64), (24, 64), (16, 48), (16, 0), (16, 544)])
def test_geometries_that_are_refused(page, d):
    with pytest.raises(ops.KernelError):
        ops.kv4_cache_shape(4, 2, page, d)


def test_tensors_off_the_device_are_refused():
    cache, table = torch.zeros(4, 2, 1, 18 * 64, dtype=torch.uint8), torch.zeros(1, 2, dtype=torch.int32)
    rows = torch.zeros(1, 2, 64)
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.kv4_write(rows, rows, None, table, cache)
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.kv4_read(cache, table, table, table, rows, rows)
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.kv4_attention(rows, rows, cache, None, table, 0, 1.0, 4, 2, 64)
