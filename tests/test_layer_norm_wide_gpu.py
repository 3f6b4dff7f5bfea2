"""GPU: rows longer than any register form takes, in 16 bits, and short rows by the lane group, against
the formulas in 64 bits (tolerances as in test_layer_norm_gpu.py)."""
import pytest
import torch

from test_layer_norm_gpu import _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("rows,width", [(3, 16385), (2, 32770), (2, 65544)])       # single values, pairs, vectors
def test_wide_rows_in_16_bits(cuda, dtype, w_dtype, rows, width):
    x, w, b, dy = _inputs(width, rows, width, dtype, w_dtype)
    _check(cuda, x, w, b, dy)


@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                           (torch.float32, torch.float32)])
@pytest.mark.parametrize("width", [8, 56, 72, 128, 248, 256])                      # 8, 16 and 32 lanes, full and not
@pytest.mark.parametrize("rows", [1, 31, 24001])                                   # more rows than one turn of the grid
def test_lane_groups(cuda, dtype, w_dtype, width, rows):
    x, w, b, dy = _inputs(width + rows, rows, width, dtype, w_dtype)
    _check(cuda, x, w, b, dy)
