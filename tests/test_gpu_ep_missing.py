"""Pairs without an expert (id -1, as the router marks padding tokens and rows with too few live experts) on the expert-parallel
layer's paths: they go nowhere, add nothing whatever their weight is, and leave every buffer outside their own alone."""
import ctypes

import pytest
import torch

import asymgemm_b200 as ag
from asymgemm_b200 import _lib, ep, moe_ops
from tests.test_gpu_ep import _make_weights

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _routed(tokens, experts, k, seed, used):
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn((tokens, experts), generator=gen)
    logits[1, 1:] = -float("inf")            # one expert left
    logits[3] = float("nan")                 # none
    rows = torch.tensor([used], dtype=torch.int32, device=DEV)
    return moe_ops.route_topk(logits.to(DEV), k, scoring="sigmoid", rows_used=rows)


@pytest.mark.parametrize("exchange", ["nccl", "peer"])
def test_layer_on_one_gpu_takes_what_the_router_gives(exchange):
    experts, hidden, inter, tokens, k, used = 8, 512, 256, 300, 3, 270
    w13, s13, w2, s2 = _make_weights(experts, hidden, inter, DEV)
    args = (experts, hidden, inter, (w13.pin_memory(), s13.to(DEV)), (w2.pin_memory(), s2.to(DEV)))
    layer = ep.ExpertParallelMoE(*args, exchange=exchange, max_tokens=tokens, top_k=k)
    try:
        gen = torch.Generator().manual_seed(60)
        x = torch.randn((tokens, hidden), generator=gen).to(torch.bfloat16).to(DEV)
        full = torch.stack([torch.randperm(experts, generator=gen)[:k] for _ in range(tokens)]).to(DEV)
        layer.forward(x, full, torch.rand((tokens, k), device=DEV))         # leaves rows, addresses and results behind
        ids, w = _routed(tokens, experts, k, 61, used)
        assert bool((ids[used:] == -1).all()) and ids[1].tolist() == [0, -1, -1] and ids[3].tolist() == [-1] * k
        y = layer.forward(x, ids, w)
        ag.check_status()
        assert float(y[used:].abs().max()) == 0 and float(y[3].abs().max()) == 0 and bool(torch.isfinite(y.float()).all())
        # the missing pairs count for nothing: any expert in their place with weight 0 gives the same, and their weight is not looked at
        plain = ep.ExpertParallelMoE(*args)
        assert torch.equal(plain.forward(x, ids.clamp(min=0), w), y)
        assert torch.equal(layer.forward(x, ids, torch.where(ids < 0, float("nan"), w)), y)
        # no pair at all
        assert float(layer.forward(x, torch.full_like(ids, -1), w).abs().max()) == 0
        assert torch.equal(layer.forward(x, ids, w), y)
    finally:
        if layer.peer is not None:
            layer.peer.close()


class _Guarded:
    """A buffer of bytes with filled margins on both sides."""

    def __init__(self, nbytes, margin=4096):
        self.all = torch.full((nbytes + 2 * margin,), 0xAB, dtype=torch.uint8, device=DEV)
        self.body, self.margin = self.all[margin:margin + nbytes], margin

    def check(self):
        assert bool((self.all[: self.margin] == 0xAB).all()) and bool((self.all[self.all.numel() - self.margin:] == 0xAB).all())


@pytest.mark.parametrize("bad", [False, True])
def test_exchange_kernels_of_two_ranks_skip_missing_pairs(bad):
    """The steps of two ranks one after the other on one GPU (no kernel of the exchange waits for another)."""
    lib = _lib.load()
    experts, k, row_bytes, ret_bytes, cap = 6, 3, 64, 32, 8 * 128
    lo, world, tokens = torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV), 2, (40, 13)
    gen = torch.Generator().manual_seed(5)
    stream = torch.cuda.current_stream().cuda_stream
    xs, ids = [], []
    for t in tokens:
        xs.append(torch.randint(0, 256, (t, row_bytes), generator=gen, dtype=torch.uint8).to(DEV))
        e = torch.stack([torch.randperm(experts, generator=gen)[:k] for _ in range(t)])
        e[torch.rand(e.shape, generator=gen) < 0.3] = -1
        e[-2:] = -1
        if bad:
            e[0, 0], e[1, 2], e[2, 1], e[3, 0] = experts, -2, (1 << 32) + 1, -(1 << 40)
        ids.append(e.to(DEV))
    sf = [torch.rand((t, 1), generator=gen).to(DEV) for t in tokens]
    live = [(e >= 0) & (e < experts) for e in ids]
    buffers = [[_Guarded(cap * row_bytes), _Guarded(cap * 4), _Guarded(cap * 8), _Guarded(tokens[r] * k * ret_bytes)] for r in range(world)]
    for b in buffers:
        b[2].body.view(torch.int64).fill_(-1)
    peers = _lib.EpPeers()
    for r in range(world):
        peers.a[r], peers.sfa[r], peers.meta[r], peers.ret[r] = (g.body.data_ptr() for g in buffers[r])
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    counts = torch.zeros((world, experts), dtype=torch.int32, device=DEV)
    for r in range(world):
        _lib.check(lib.ag_ep_histogram(ids[r].data_ptr(), ids[r].numel(), experts, counts[r].data_ptr(), status.data_ptr(), stream))
        assert counts[r].tolist() == torch.bincount(ids[r][live[r]], minlength=experts).tolist()
    tables = []
    for r in range(world):
        # tables with margins of their own: a slot counter or a first row is never looked up for a missing expert
        send_base, cursors = _Guarded(experts * 4), _Guarded(experts * 4)
        offsets, segs = torch.zeros(8, dtype=torch.int32, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV)
        used = torch.zeros(2, dtype=torch.int32, device=DEV)
        _lib.check(lib.ag_ep_plan(counts.data_ptr(), lo.data_ptr(), world, r, experts, cap, send_base.body.data_ptr(), cursors.body.data_ptr(), offsets.data_ptr(),
                                  segs.data_ptr(), 4, used.data_ptr(), buffers[r][2].body.data_ptr(), status.data_ptr(), stream))
        tables.append((send_base, cursors, used))
    pair_rows = []
    for r in range(world):
        pair_row = torch.full((ids[r].numel(),), -9, dtype=torch.int64, device=DEV)
        _lib.check(lib.ag_ep_dispatch(xs[r].data_ptr(), sf[r].data_ptr(), ids[r].data_ptr(), tokens[r], k, row_bytes, 1, lo.data_ptr(), world, r,
                                      tables[r][0].body.data_ptr(), tables[r][1].body.data_ptr(), cap, pair_row.data_ptr(), ctypes.byref(peers), stream))
        assert torch.equal(pair_row >= 0, live[r].view(-1)) and bool((pair_row[pair_row < 0] == -1).all())
        assert torch.equal(tables[r][1].body.view(torch.int32), counts[r])
        pair_rows.append(pair_row)
    for r in range(world):
        out = buffers[r][0].body.view(cap, row_bytes)[:, :ret_bytes].contiguous()      # stands in for the experts
        _lib.check(lib.ag_ep_return(out.data_ptr(), buffers[r][2].body.data_ptr(), tables[r][2].data_ptr(), cap, ret_bytes, world, ctypes.byref(peers), stream))
    for r in range(world):
        back = buffers[r][3].body.view(tokens[r] * k, ret_bytes)
        flat, want = live[r].view(-1), xs[r][:, :ret_bytes].repeat_interleave(k, 0)
        assert torch.equal(back[flat], want[flat]) and bool((back[~flat] == 0xAB).all())
        owner = (ids[r].view(-1) >= 2).long()
        for o in range(world):
            sel = flat & (owner == o)
            assert torch.equal(buffers[o][0].body.view(cap, row_bytes)[pair_rows[r][sel]], xs[r].repeat_interleave(k, 0)[sel])
            assert torch.equal(buffers[o][1].body.view(torch.float32)[pair_rows[r][sel]], sf[r].view(-1).repeat_interleave(k)[sel])
        for g in buffers[r] + list(tables[r][:2]):
            g.check()
    assert int(status) == (_lib.EP_BAD_EXPERT if bad else 0)


def test_pairs_without_room_are_left_out_of_the_combine():
    """One rank whose buffers are too small: reported, and every pair either has a row of its own or none."""
    lib = _lib.load()
    experts, k, tokens, cap = 2, 1, 300, 256
    x, sf = torch.randint(0, 256, (tokens, 64), dtype=torch.uint8, device=DEV), torch.rand((tokens, 1), device=DEV)
    ids = torch.zeros((tokens, k), dtype=torch.int64, device=DEV)
    a, s, meta, ret = _Guarded(cap * 64), _Guarded(cap * 4), _Guarded(cap * 8), _Guarded(64)
    peers = _lib.EpPeers()
    peers.a[0], peers.sfa[0], peers.meta[0], peers.ret[0] = (g.body.data_ptr() for g in (a, s, meta, ret))
    lo = torch.tensor([0, experts], dtype=torch.int32, device=DEV)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)
    status, counts, send_base, cursors, offsets, segs, used = i32(1), i32(experts), i32(experts), i32(experts), i32(4), i32(3), i32(2)
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.ag_ep_histogram(ids.data_ptr(), tokens, experts, counts.data_ptr(), status.data_ptr(), stream))
    _lib.check(lib.ag_ep_plan(counts.data_ptr(), lo.data_ptr(), 1, 0, experts, cap, send_base.data_ptr(), cursors.data_ptr(), offsets.data_ptr(), segs.data_ptr(),
                              2, used.data_ptr(), meta.body.data_ptr(), status.data_ptr(), stream))
    pair_row = torch.full((tokens,), -9, dtype=torch.int64, device=DEV)
    _lib.check(lib.ag_ep_dispatch(x.data_ptr(), sf.data_ptr(), ids.data_ptr(), tokens, k, 64, 1, lo.data_ptr(), 1, 0, send_base.data_ptr(), cursors.data_ptr(), cap,
                                  pair_row.data_ptr(), ctypes.byref(peers), stream))
    assert int(status) == _lib.EP_OVERFLOW
    kept = pair_row >= 0
    assert sorted(pair_row[kept].tolist()) == list(range(cap)) and bool((pair_row[~kept] == -1).all())
    assert torch.equal(a.body.view(cap, 64)[pair_row[kept]], x[kept])
    for g in (a, s, meta, ret):
        g.check()


@pytest.mark.parametrize("experts,dtype", [(1100, torch.int64), (6, torch.int16), (6, torch.int64)])
def test_dispatcher_on_one_gpu_without_and_with_the_layout_kernels(experts, dtype):
    """More experts than the layout kernels take, and ids of a type that they do not: laid out by torch, without a host wait."""
    tokens, k, cols = 50, 3, 64
    gen = torch.Generator().manual_seed(70)
    ids = torch.randint(0, experts, (tokens, k), generator=gen)
    ids[torch.rand(ids.shape, generator=gen) < 0.3] = -1
    ids[40:] = -1
    x = torch.randn((tokens, cols), generator=gen).to(torch.bfloat16)
    w = torch.rand((tokens, k), generator=gen)
    w[ids < 0] = float("nan")
    disp = ep.EPDispatcher(experts)
    state, recv, _ = disp.dispatch(x.to(DEV), ids.to(dtype).to(DEV))
    want_state, want_recv, _ = ep.EPDispatcher(experts).dispatch(x, ids)
    assert (state.tables is None) == (experts > 1024 or dtype == torch.int16)
    a, want_a = ep.to_contiguous_layout(recv, state), ep.to_contiguous_layout(want_recv, want_state)
    assert torch.equal(a.cpu(), want_a) and torch.equal(state.offsets.cpu(), want_state.offsets)
    y = disp.combine(a, state, w.to(DEV)).cpu()
    want = torch.where(ids < 0, 0, w).double().sum(1, keepdim=True) * x.double()
    # k products and additions in fp32, one rounding to bf16
    assert bool(((y.double() - want).abs() <= want.abs() * (2 ** -8 + 2 * k * 2 ** -24)).all())


@pytest.mark.expects_status
@pytest.mark.parametrize("experts", [6, 1100])
def test_ids_outside_the_experts_are_dropped_and_reported_by_the_dispatcher(experts):
    ids = torch.tensor([[0, experts], [-2, 1], [3, -1]], device=DEV)
    x = torch.ones((3, 64), dtype=torch.bfloat16, device=DEV)
    disp = ep.EPDispatcher(experts)
    state, recv, _ = disp.dispatch(x, ids)
    assert int(state.rows_per_expert.sum()) == 3
    y = disp.combine(ep.to_contiguous_layout(recv, state), state, torch.ones((3, 2), device=DEV))
    assert y[:, 0].tolist() == [1.0, 1.0, 1.0]
    with pytest.raises(RuntimeError, match="expert id"):
        ag.check_status()
    ag.check_status()


@pytest.mark.parametrize("missing", [0.0, 0.3, 1.0])
def test_the_state_of_one_gpu_has_the_sort_that_the_cpu_has(missing):
    tokens, experts, k = 43, 7, 3
    gen = torch.Generator().manual_seed(80)
    ids = torch.stack([torch.randperm(experts, generator=gen)[:k] for _ in range(tokens)])
    ids[torch.rand(ids.shape, generator=gen) < missing] = -1
    x = torch.randn((tokens, 8), generator=gen)
    gpu, _, _ = ep.EPDispatcher(experts).dispatch(x.to(DEV), ids.to(DEV))
    cpu, _, _ = ep.EPDispatcher(experts).dispatch(x, ids)
    assert isinstance(gpu, ep.DispatchState) and gpu.tables is not None
    for name in ("order", "dest_rows", "src_token"):
        assert torch.equal(getattr(gpu, name).cpu(), getattr(cpu, name)), name
    assert gpu.send_splits == cpu.send_splits and gpu.recv_splits == cpu.recv_splits and gpu.padded_rows == cpu.padded_rows
