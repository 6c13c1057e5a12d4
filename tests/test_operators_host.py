"""Host side of the operators around the grouped GEMMs: routings that name no expert, tensors that are not on a GPU, empty inputs.
No GPU is needed."""
import types

import pytest
import torch

from asymgemm_b200 import ep_peer


@pytest.mark.parametrize("world", [1, 2])
def test_peer_exchange_reads_no_result_of_a_pair_that_was_sent_nowhere(world):
    went = torch.tensor([7, -1, 0, 130, -1, 2, 99, 99])      # longer than the step's six pairs
    px = types.SimpleNamespace(pair_row=went, world=world, _ids=torch.zeros((3, 2)), _slots=torch.arange(8))
    rows = ep_peer.PeerExchange.result_rows(px)
    assert rows.tolist() == ([7, -1, 0, 130, -1, 2] if world == 1 else [0, -1, 2, 3, -1, 5])
