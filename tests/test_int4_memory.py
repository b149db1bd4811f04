"""What the kernels read of a 4-bit weight lies within its tensors' memory, without a GPU."""

import pytest
import torch

from feather_ops import int4


def _strided(rows, groups, offset, pitch, room, dtype):
    """[rows, groups] stored group by group in a storage that ends `room` values behind the last one."""
    size = offset + (groups - 1) * pitch + rows + room
    return torch.arange(size).to(dtype).as_strided((rows, groups), (1, pitch), offset)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8])
@pytest.mark.parametrize("rows,groups,pitch", [(1, 1, 4), (1, 3, 4), (2, 2, 6), (3, 2, 4), (3, 1, 8), (4, 2, 4), (5, 3, 5), (9, 2, 12)])
def test_groups_of_scales(rows, groups, pitch, dtype):
    """4 values of each group are read, its last 4 or, of fewer, what lies behind them."""
    for offset in (0, 3):
        for room in range(4):
            t = _strided(rows, groups, offset, pitch, room, dtype)
            got = int4._grouped(t)
            assert torch.equal(got, t)
            step = got.stride(1) if groups > 1 else max(rows, got.stride(1))
            assert (rows == 1 or got.stride(0) == 1) and step >= max(rows, 4)
            end = got.storage_offset() + (groups - 1) * got.stride(1) + max(rows, 4)
            assert end * got.element_size() <= got.untyped_storage().nbytes()
            if rows >= 4 or room >= 4 - rows:
                assert got is t   # not copied where it need not be


@pytest.mark.parametrize("rows,cols,pitch", [(1, 1, 1), (1, 7, 7), (3, 5, 8), (4, 8, 8), (2, 3, 4), (5, 9, 12)])
def test_rows_of_codes(rows, cols, pitch):
    """Each row is read to a multiple of 4 bytes."""
    for offset in (0, 4, 2):
        for room in range(4):
            size = offset + (rows - 1) * pitch + cols + room
            t = torch.arange(size).to(torch.uint8).as_strided((rows, cols), (pitch, 1), offset)
            got = int4._whole_bytes(t)
            assert torch.equal(got, t) and got.storage_offset() % 4 == 0 and (rows == 1 or got.stride(0) % 4 == 0)
            end = got.storage_offset() + (rows - 1) * got.stride(0) + -(-cols // 4) * 4
            assert end <= got.untyped_storage().nbytes()
