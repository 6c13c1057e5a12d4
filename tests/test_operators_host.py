"""Host side of the operators around the grouped GEMMs: routings that name no expert, tensors that are not on a GPU, empty inputs.
No GPU is needed."""
import types

import pytest
import torch

from asymgemm_b200 import api, dense_ops, ep_peer, moe_ops
from asymgemm_b200.ep import EPDispatcher, to_contiguous_layout
from tests import test_ep_gloo as gloo


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


@pytest.mark.parametrize("dtype", [torch.float32, torch.float8_e4m3fn])
def test_cpu_row_moves_with_and_without_a_destination(dtype):
    src = torch.arange(30, dtype=torch.float32).view(6, 5).to(dtype)
    dst = torch.tensor([2, -1, 0, -5, 3, 9])
    out = moe_ops.move_rows(src, 4, dst_rows=dst, count=5, zero=True)
    want = torch.stack([src[2], torch.zeros(5).to(dtype), src[0], src[4]])
    assert out.shape == (4, 5) and out.dtype == dtype and torch.equal(out.float(), want.float())
    out = moe_ops.move_rows(src, 4, src_rows=torch.tensor([5, -1, 1, 0, 3, 3]), dst_rows=dst, count=5, zero=True)
    want = torch.stack([src[1], torch.zeros(5).to(dtype), src[5], src[3]])
    assert torch.equal(out.float(), want.float())
    out = moe_ops.move_rows(src, 4, src_rows=torch.tensor([5, -1, 1]), count=2, zero=True)
    assert torch.equal(out[0].float(), src[5].float()) and float(out[1:].float().abs().max()) == 0


def test_cpu_combine_does_not_look_at_the_weight_of_a_missing_row():
    rows = torch.arange(12.0).view(4, 3)
    rows[0] = float("inf")
    a, w = rows.requires_grad_(True), torch.tensor([[0.5, float("nan")], [float("inf"), 2.0]], requires_grad=True)
    y = moe_ops.combine_topk(a, torch.tensor([1, -1, -1, 3]), w, 2, 2)
    assert torch.equal(y, torch.stack([0.5 * rows[1], 2 * rows[3]]))
    da, dw = torch.autograd.grad(y, (a, w), torch.ones(2, 3))
    assert da.tolist() == [[0.0] * 3, [0.5] * 3, [0.0] * 3, [2.0] * 3]
    assert dw.tolist() == [[float(rows[1].detach().sum()), 0.0], [0.0, float(rows[3].detach().sum())]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_cpu_combine_takes_a_table_longer_than_the_batch(dtype):
    rows, w = torch.arange(12.0).view(4, 3).to(dtype), torch.tensor([[0.5, 1.0], [0.25, 2.0]])
    short = torch.tensor([3, 0, -1, 2])
    want = moe_ops.combine_topk(rows, short, w, 2, 2)
    assert torch.equal(moe_ops.combine_topk(rows, torch.cat([short, torch.tensor([1, 1, -1])]), w, 2, 2), want)
    assert torch.equal(moe_ops.combine_topk(rows, short.view(2, 2), w, 2, 2), want)


# ------------------------------------------------------------------------------------------------------ exchange between ranks
def _missing_ids(rank, tokens, experts, k):
    """What the router gives: -1 where a row has too few live experts and in the padding tokens at the end; rank 2 has nothing else."""
    gen = torch.Generator().manual_seed(200 + rank)
    ids = torch.stack([torch.randperm(experts, generator=gen)[:k] for _ in range(tokens)])
    ids[torch.rand(ids.shape, generator=gen) < 0.2] = -1
    ids[tokens - 5:] = -1
    return torch.full_like(ids, -1) if rank == 2 else ids


def _missing_worker(rank, world, port, q):
    try:
        gloo._init(rank, world, port)
        experts, tokens, hidden, k = 12, 31 + 4 * rank, 16, 3
        x = torch.randn((tokens, hidden), generator=torch.Generator().manual_seed(rank))
        x[tokens - 5:] = float("nan")
        ids = _missing_ids(rank, tokens, experts, k)
        w = torch.rand((tokens, k), generator=torch.Generator().manual_seed(50 + rank))
        w[ids < 0] = float("nan")
        want = torch.where(ids < 0, 0, (ids + 1).float() * w).sum(dim=1, keepdim=True) * torch.nan_to_num(x)
        tag = torch.arange(tokens, dtype=torch.float32).unsqueeze(1)
        disp = EPDispatcher(experts)
        first = disp.expert_ranges[rank][0]
        state, recv, (recv_tag,) = disp.dispatch(x, ids, (tag,))
        assert sum(state.send_splits) == int((ids >= 0).sum()) and recv.shape[0] == recv_tag.shape[0] == int(state.rows_per_expert.sum()) == sum(state.recv_splits)
        y = disp.combine(gloo._fake_experts(to_contiguous_layout(recv, state), state, first), state, w)
        assert torch.allclose(y, want, rtol=1e-5, atol=1e-5), (y - want).abs().max()
        for groups in (1, 2, 3):
            def group_fn(rows, extras, st, start, count):
                return gloo._fake_experts(to_contiguous_layout(rows, st), st, first + start)

            y = disp.pipelined(x, (tag,), ids, w, groups, group_fn)
            assert torch.allclose(y, want, rtol=1e-5, atol=1e-5), (groups, (y - want).abs().max())
        torch.distributed.barrier()
        q.put((rank, "ok"))
    except Exception as e:  # pragma: no cover - reported through the queue
        q.put((rank, f"error: {type(e).__name__}: {e}"))
    finally:
        if torch.distributed.is_initialized():
            torch.distributed.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_ranks_exchange_no_row_for_pairs_without_an_expert(world):
    results = gloo._run(_missing_worker, world=world)
    assert results == {r: "ok" for r in range(world)}, results


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16])
def test_one_rank_gives_pairs_without_an_expert_no_row(dtype):
    disp = EPDispatcher(4)
    ids = torch.tensor([[0, 3], [-1, 1], [3, -1], [-1, -1]], dtype=dtype)
    x = torch.arange(4, dtype=torch.float32).unsqueeze(1) + 1
    state, recv, _ = disp.dispatch(x, ids)
    assert state.rows_per_expert.tolist() == [1, 1, 0, 2]
    a = to_contiguous_layout(recv, state)
    assert a[0, 0] == 1 and a[128, 0] == 2 and a[256:258, 0].tolist() == [1.0, 3.0] and float(a.abs().sum()) == 7
    w = torch.tensor([[1.0, 1.0], [float("nan"), 1.0], [1.0, float("inf")], [float("nan")] * 2])
    assert disp.combine(a, state, w).view(-1).tolist() == [2.0, 2.0, 3.0, 0.0]
    state, recv, _ = disp.dispatch(x, torch.full_like(ids, -1))
    a = to_contiguous_layout(recv, state)
    assert float(a.abs().sum()) == 0 and float(disp.combine(a, state, w).abs().sum()) == 0
    for bad in (4, -2, 100):
        ids[1, 1] = bad
        with pytest.raises(RuntimeError, match="expert id"):
            disp.dispatch(x, ids)


def test_a_refused_cpu_tensor_leaves_no_status_word_behind(monkeypatch):
    """The words are kept by GPU index, which a CPU tensor does not have: it must not become the current GPU's."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(api, "_status_cache", {})
    x, ids = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((4, 2), dtype=torch.int64)
    for call in (lambda: dense_ops.linear(x, x), lambda: dense_ops.linear_backward(x, x, x), lambda: moe_ops.route_layout(ids, 8),
                 lambda: moe_ops.route_layout_masked(ids, 8, 4), lambda: moe_ops.combine_topk_backward(x, x, None, torch.zeros(4, 1))):
        with pytest.raises(RuntimeError):
            call()
        assert not api._status_cache
