"""Host side of the operators around the grouped GEMMs: routings that name no expert, tensors that are not on a GPU, empty inputs.
No GPU is needed."""
import types

import pytest
import torch

from asymgemm_b200 import ep_peer, moe_ops


@pytest.mark.parametrize("world", [1, 2])
def test_peer_exchange_reads_no_result_of_a_pair_that_was_sent_nowhere(world):
    went = torch.tensor([7, -1, 0, 130, -1, 2, 99, 99])      # longer than the step's six pairs
    px = types.SimpleNamespace(pair_row=went, world=world, _ids=torch.zeros((3, 2)), _slots=torch.arange(8))
    rows = ep_peer.PeerExchange.result_rows(px)
    assert rows.tolist() == ([7, -1, 0, 130, -1, 2] if world == 1 else [0, -1, 2, 3, -1, 5])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn])
def test_tables_of_missing_rows_read_nothing_where_there_are_no_rows(dtype):
    src, none = torch.zeros((0, 16), dtype=dtype), torch.full((6,), -1)
    out = moe_ops.move_rows(src, 6, src_rows=none)
    assert out.dtype == dtype and out.shape == (6, 16) and not out.view(torch.uint8).any()
    out = moe_ops.move_rows(src, 4, src_rows=none[:2], dst_rows=torch.tensor([3, -1]), zero=True)
    assert out.shape == (4, 16) and not out.view(torch.uint8).any()
    if dtype != torch.float8_e4m3fn:
        leaf = src.clone().requires_grad_(True)
        y = moe_ops.combine_topk(leaf, none, torch.ones(3, 2), 3, 2)
        assert y.shape == (3, 16) and y.dtype == dtype and float(y.detach().abs().max()) == 0
        assert torch.autograd.grad(y.sum(), leaf)[0].shape == (0, 16)
