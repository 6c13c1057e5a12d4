"""Operators around the grouped GEMMs where calls are unusual: nothing to do, tables longer than the batch, widths and types without
a kernel, calls recorded into graphs, derivatives that are not there."""
import math

import pytest
import torch

import asymgemm_b200 as ag
from asymgemm_b200 import moe_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


@pytest.mark.parametrize("cols", [64, 12, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
def test_an_empty_batch_in_the_masked_layout(cols, dtype):
    lay = moe_ops.route_layout_masked(torch.zeros((0, 2), dtype=torch.int64, device=DEV), 4, 8)
    x = torch.empty((0, cols), dtype=dtype, device=DEV)
    out = moe_ops.move_rows(x, lay.row_token.numel(), src_rows=lay.row_token)
    assert out.shape == (32, cols) and float(out.float().abs().max()) == 0
    y = moe_ops.combine_topk(x, torch.full((6,), -1, device=DEV), torch.ones((3, 2), device=DEV), 3, 2)
    assert y.shape == (3, cols) and float(y.float().abs().max()) == 0
