"""Tokens behind a block's size are no keys: their gradients are zero, whatever the rows that attend to the block hold."""
import math

import pytest
import torch

from tests.helpers import dev
from tests.test_selected_attention import _inputs, _run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,block", [(torch.bfloat16, 128, 64), (torch.bfloat16, 128, 128), (torch.float32, 128, 64), (torch.float32, 40, 16), (torch.float32, 200, 32)])
@pytest.mark.parametrize("which", ["query", "dout", "value"])
def test_no_number_in_a_row_that_attends(dtype, D, block, which):
    g = torch.Generator(device=dev()).manual_seed(block)
    Lq, Lkv, H, Hkv = 2 * block + 5, 5 * block - 3, 4, 2
    q, k, v, dout = _inputs(g, 1, Lq, Lkv, H, Hkv, D, dtype)
    index = torch.tensor([[0, 2, 4], [2, 1, 0], [4, 0, 1]], dtype=torch.int32, device=dev()).expand(1, H, 3, 3).contiguous()
    num = torch.full((1, H, 3), 3, dtype=torch.int32, device=dev())
    sizes = torch.tensor([block - 3, block // 2, 1, 4, block], dtype=torch.int32, device=dev())
    {"query": q, "dout": dout, "value": v}[which][0, 0] = math.nan
    got = _run(q, k, v, index, num, block, dout, block_sizes=sizes)
    at = torch.arange(Lkv, device=dev())
    behind = at % block >= sizes[at // block]
    assert int(behind.sum()) > block and bool(torch.isnan(got["dk"][:, ~behind]).any())
    assert not bool(got["dk"][:, behind].any()) and not bool(got["dv"][:, behind].any())      # (a NaN counts as true)
