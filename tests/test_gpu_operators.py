"""Operators around the grouped GEMMs where calls are unusual: nothing to do, tables longer than the batch, widths and types without
a kernel, calls recorded into graphs, derivatives that are not there."""
import subprocess
import sys

import pytest
import torch

import asymgemm_b200 as ag
from asymgemm_b200 import dense_ops, moe_ops

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


@pytest.mark.parametrize("cols,dtype", [(5, torch.float32), (18, torch.float32), (12, torch.bfloat16), (40, torch.float8_e4m3fn), (64, torch.bfloat16)])
def test_row_moves_without_a_kernel_do_not_wait_for_the_device(cols, dtype):
    """Rows whose bytes are no multiple of 16 (scale rows of some widths): a call that waited could not be captured."""
    src = randn(50, cols, seed=1).to(dtype)
    gen = torch.Generator().manual_seed(2)
    dst = torch.randperm(60, generator=gen)[:50]
    dst[::7] = -1
    pick = torch.randint(-1, 50, (50,), generator=gen)
    dst, pick = dst.to(DEV), pick.to(DEV)
    moe_ops.move_rows(src, 60, src_rows=pick, dst_rows=dst, zero=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = moe_ops.move_rows(src, 60, src_rows=pick, dst_rows=dst, zero=True)
    src.copy_(randn(50, cols, seed=3).to(dtype))
    graph.replay()
    want = torch.zeros((60, cols), dtype=torch.float64)
    for i, (d, s) in enumerate(zip(dst.tolist(), pick.tolist())):
        if d >= 0 and s >= 0:
            want[d] = src[s].cpu().double()
    assert out.shape == (60, cols) and out.dtype == dtype and torch.equal(out.float().cpu().double(), want)


@pytest.mark.parametrize("dtype,cols", [(torch.bfloat16, 64), (torch.float32, 64), (torch.float32, 12), (torch.float16, 64), (torch.bfloat16, 12), (torch.float32, 5)])
def test_the_combine_of_an_empty_batch_has_the_type_of_any_other(dtype, cols):
    rows, pos, w = randn(8, cols, seed=4, dtype=dtype), torch.arange(8, device=DEV), torch.rand((4, 2), device=DEV)
    for fn in (moe_ops.combine_topk, moe_ops.combine_topk_forward):
        full, empty = fn(rows, pos, w, 4, 2), fn(rows, pos[:0], w[:0], 0, 2)
        assert empty.shape == (0, cols) and empty.dtype == full.dtype


@pytest.mark.parametrize("dtype,cols", [(torch.bfloat16, 64), (torch.float32, 64), (torch.float32, 12), (torch.float16, 64)])
def test_combine_without_a_position_table(dtype, cols):
    rows, w = randn(14, cols, seed=5, dtype=dtype), torch.rand((4, 3), device=DEV)
    y = moe_ops.combine_topk(rows, None, w, 4, 3)
    assert torch.equal(y, moe_ops.combine_topk(rows, torch.arange(12, device=DEV), w, 4, 3))
    want = (rows[:12].double().view(4, 3, cols) * w.double().unsqueeze(2)).sum(1)
    size = (rows[:12].double().view(4, 3, cols) * w.double().unsqueeze(2)).abs().sum(1)
    # three products and additions in fp32, one rounding
    assert bool(((y.double() - want).abs() <= size * 6 * 2 ** -24 + want.abs() * torch.finfo(y.dtype).eps / 2).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_combine_refuses_tables_that_its_kernels_would_read_past(dtype):
    rows, pos, w = randn(16, 64, seed=6, dtype=dtype), torch.arange(12, device=DEV), torch.rand((6, 2), device=DEV)
    want = moe_ops.combine_topk(rows, pos, w, 6, 2)
    for bad in ((rows, pos.int(), w), (rows, pos[:11], w), (rows, pos.cpu(), w), (rows, torch.arange(24, device=DEV)[::2], w), (rows, pos, w[:5]), (rows, pos, w.cpu()),
                (rows[:11], None, w)):
        for grad in (False, True):
            with pytest.raises(RuntimeError):
                moe_ops.combine_topk(bad[0].clone().requires_grad_(grad), bad[1], bad[2], 6, 2)
    assert torch.equal(moe_ops.combine_topk(rows, pos.view(6, 2), w, 6, 2), want)
    assert torch.equal(moe_ops.combine_topk(rows, pos, torch.cat([w, w]), 6, 2), want)


@pytest.mark.parametrize("cols", [4, 12, 20, 1028])
@pytest.mark.parametrize("table", [True, False])
def test_gradient_of_the_combine_at_widths_where_only_the_sum_has_a_kernel(cols, table):
    """fp32 rows of 4 mod 8 columns."""
    tokens, k = 7, 3
    rows, w = randn(40, cols, seed=7), torch.rand((tokens, k), generator=torch.Generator().manual_seed(8)).to(DEV)
    pos = torch.randperm(40, generator=torch.Generator().manual_seed(9))[: tokens * k].to(DEV) if table else None
    if table:
        pos[::5] = -1
    dy = randn(tokens, cols, seed=10, dtype=torch.bfloat16)
    a, b = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = moe_ops.combine_topk(a, pos, b, tokens, k)
    assert torch.equal(y.detach(), moe_ops.combine_topk(rows, pos, w, tokens, k))
    drows, dweights = torch.autograd.grad(y, (a, b), dy, retain_graph=True)
    at = pos if table else torch.arange(tokens * k, device=DEV)
    live = at >= 0
    g = dy.double().repeat_interleave(k, 0)
    want = torch.zeros(rows.shape, dtype=torch.float64, device=DEV)
    want[at[live]] = (w.double().view(-1, 1) * g)[live]
    assert drows.dtype == torch.float32 and bool(((drows.double() - want).abs() <= want.abs() * 2 ** -23).all())
    terms = torch.where(live.unsqueeze(1), rows.double()[at.clamp(min=0)] * g, 0)
    # a product and at most `cols` additions in fp32
    assert bool(((dweights.double().view(-1) - terms.sum(1)).abs() <= terms.abs().sum(1) * (cols + 1) * 2 ** -24).all())
    assert torch.equal(torch.autograd.grad(y, a, dy, retain_graph=True)[0], drows) and torch.equal(torch.autograd.grad(y, b, dy)[0], dweights)
    assert torch.equal(torch.autograd.grad(moe_ops.combine_topk(rows, pos, b, tokens, k), b, dy)[0], dweights)
    assert torch.equal(torch.autograd.grad(moe_ops.combine_topk(a, pos, w, tokens, k), a, dy)[0], drows)
    empty = moe_ops.combine_topk(a, None if pos is None else pos[:0], b[:0], 0, k)
    assert empty.shape == (0, cols) and float(torch.autograd.grad(empty.sum(), a)[0].abs().max()) == 0


LAYOUTS_AT_THE_SHARED_MEMORY_LIMIT = """
import threading, torch
import asymgemm_b200 as ag
from asymgemm_b200 import dense_ops, moe_ops

def check(tokens, experts):
    ids = torch.randint(-1, experts, (tokens, 2), generator=torch.Generator().manual_seed(experts))
    got = moe_ops.route_layout(ids.cuda(), experts, 1)
    flat = ids.view(-1)
    order = torch.argsort(torch.where(flat < 0, experts, flat), stable=True)[: int((flat >= 0).sum())]
    want = torch.full((flat.numel(),), -1)
    want[order] = torch.arange(order.numel())
    assert torch.equal(got.pair_row.cpu(), want), (tokens, experts)
    assert torch.equal(got.rows_per_expert.cpu(), torch.bincount(flat[flat >= 0], minlength=experts)), (tokens, experts)

for tokens in (700, 2500):          # one block, several
    for experts in (351, 350, 352, 1024, 351):
        check(tokens, experts)
failed = []
def many(experts):
    try:
        for _ in range(60):
            check(700, experts)
            check(2500, experts)
    except Exception as e:
        failed.append((experts, repr(e)))
threads = [threading.Thread(target=many, args=(e,)) for e in (360, 1024, 500, 20)]
for t in threads: t.start()
for t in threads: t.join()
assert not failed, failed
ag.check_status()
print("done")
"""


def test_layouts_at_the_limit_of_shared_memory_and_from_several_threads():
    """In a process of its own: 351 experts, whose tables just pass the default limit together with the kernel's own, come first."""
    res = subprocess.run([sys.executable, "-c", LAYOUTS_AT_THE_SHARED_MEMORY_LIMIT], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip() == "done", res.stdout + res.stderr


def test_forward_mode_derivatives_are_refused_or_right():
    """A tangent is never dropped in silence."""
    from torch.autograd import forward_ad
    x, w, g = randn(8, 64, seed=11, dtype=torch.bfloat16), randn(16, 64, seed=12, dtype=torch.bfloat16), randn(8, 16, seed=13, dtype=torch.bfloat16)
    logits, dw, bias = randn(8, 16, seed=14), randn(8, 2, seed=15), randn(16, seed=16)
    ids, _ = moe_ops.route_topk(logits, 2)
    rows, pos, weights = randn(16, 64, seed=17, dtype=torch.bfloat16), torch.randperm(16, device=DEV), torch.rand((8, 2), device=DEV)
    pos[3] = -1
    dy = randn(8, 64, seed=18, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: moe_ops.route_topk(dual(logits), 2), lambda: moe_ops.route_topk(logits, 2, bias=dual(bias)),
                     lambda: moe_ops.route_topk(dual(logits.clone().requires_grad_(True)), 2),
                     lambda: moe_ops.route_topk_backward(dual(dw), ids, logits), lambda: moe_ops.route_topk_backward(dw, ids, dual(logits)),
                     lambda: dense_ops.linear(dual(x), w), lambda: dense_ops.linear(x, dual(w)), lambda: dense_ops.linear(x, w, bias=dual(bias)),
                     lambda: dense_ops.linear(x, w, residual=dual(g)), lambda: dense_ops.linear(dual(x), w.clone().requires_grad_(True)),
                     lambda: dense_ops.linear(dual(x.view(2, 4, 64)), w), lambda: dense_ops.linear_backward(dual(g), x, w), lambda: dense_ops.linear_backward(g, dual(x), w),
                     lambda: dense_ops.linear_backward(g, x, w, activation="relu", pre=dual(g)),
                     lambda: moe_ops.combine_topk_backward(dual(dy), rows, pos, weights), lambda: moe_ops.combine_topk_backward(dy, dual(rows), pos, weights)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
        for a, b in ((dual(rows), weights), (rows, dual(weights)), (dual(rows), dual(weights))):
            y, tangent = forward_ad.unpack_dual(moe_ops.combine_topk(a, pos, b, 8, 2))
            assert y.dtype == torch.bfloat16
            live, at = (pos >= 0).view(8, 2, 1), pos.clamp(min=0)
            r, ws = rows.double()[at].view(8, 2, 64), weights.double().unsqueeze(2)
            want = (torch.where(live, ws, 0).expand_as(r) * (a is not rows) + torch.where(live, r, 0) * (b is not weights))
            # three roundings to bf16 at most (the tangents' own, the sum's) and fp32 sums of two
            assert bool(((tangent.double() - want.sum(1)).abs() <= want.abs().sum(1) * (3 * 2 ** -8)).all())
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: moe_ops.route_topk(t, 2)[1], (logits,), (torch.ones_like(logits),))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: dense_ops.linear(t, w), (x,), (torch.ones_like(x),))
    # outside of all that the calls are what they were
    assert torch.equal(moe_ops.route_topk(logits, 2)[0], ids)


def test_tables_of_one_allocation_do_not_overlap():
    for tokens, experts, k in ((1, 3, 1), (37, 60, 5), (700, 16, 3)):
        ids, weights = moe_ops.route_topk(randn(tokens, experts, seed=20), k)
        for tables in ((ids, weights), tuple(moe_ops.route_layout(ids, experts)), tuple(moe_ops.route_layout_masked(ids, experts, 7))):
            before = [t.clone() for t in tables]
            for i, t in enumerate(tables):
                t.fill_(-77)
                assert all(torch.equal(a, b) for j, (a, b) in enumerate(zip(tables, before)) if j != i)
                t.copy_(before[i])


def test_expanded_operands():
    """One row or one block of rows under many indices: the strides of the rows are 0 or shorter than a row."""
    x, w = randn(1, 64, seed=21, dtype=torch.bfloat16), randn(24, 64, seed=22, dtype=torch.bfloat16)
    r, g = randn(1, 24, seed=23, dtype=torch.bfloat16), randn(10, 24, seed=24, dtype=torch.bfloat16)
    many = lambda t, *shape: t.expand(*shape)
    y, pre = dense_ops.linear(many(x, 10, 64), w, activation="silu", residual=many(r, 10, 24), return_pre=True)
    want, want_pre = dense_ops.linear(x.repeat(10, 1), w, activation="silu", residual=r.repeat(10, 1), return_pre=True)
    assert torch.equal(y, want) and torch.equal(pre, want_pre)
    y = dense_ops.linear(many(x, 2, 5, 64), w, residual=many(r, 2, 5, 24))
    assert torch.equal(y.view(10, 24), dense_ops.linear(x.repeat(10, 1), w, residual=r.repeat(10, 1)))
    got = dense_ops.linear_backward(g, many(x, 10, 64), w, activation="silu", pre=many(pre[:1], 10, 24))
    want = dense_ops.linear_backward(g, x.repeat(10, 1), w, activation="silu", pre=pre[:1].repeat(10, 1))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = dense_ops.linear_backward(many(r, 10, 24), x.repeat(10, 1), w)
    assert all(torch.equal(a, b) for a, b in zip(got, dense_ops.linear_backward(r.repeat(10, 1), x.repeat(10, 1), w)))
    assert torch.equal(dense_ops.linear(x, many(w[:1], 9, 64)), dense_ops.linear(x, w[:1].repeat(9, 1)))
    # broadcast leaves get the sum over their copies
    leaf, shared = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
    dx, dr = torch.autograd.grad(dense_ops.linear(many(leaf, 10, 64), w, residual=many(shared, 10, 24)), (leaf, shared), g)
    rows = dense_ops.linear_backward(g, x.repeat(10, 1), w)[0].double()
    # ten rows of bf16 numbers summed by torch in fp32 at least, rounded once
    for a, b in ((dx, rows), (dr, g.double())):
        assert bool(((a.double() - b.sum(0)).abs() <= b.abs().sum(0) * 16 * 2 ** -24 + b.sum(0).abs() * 2 ** -8).all())
    logits = randn(1, 16, seed=25)
    ids, weights = moe_ops.route_topk(many(logits, 7, 16), 3, scoring="sigmoid")
    want = moe_ops.route_topk(logits.repeat(7, 1), 3, scoring="sigmoid")
    assert torch.equal(ids, want[0]) and torch.equal(weights, want[1])
    dw = randn(7, 3, seed=26)
    assert torch.equal(moe_ops.route_topk_backward(dw, ids, many(logits, 7, 16)), moe_ops.route_topk_backward(dw, ids, logits.repeat(7, 1)))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_router_gradient_leaves_out_switched_off_experts_whatever_their_gradient(scoring, renormalize):
    logits = randn(4, 40, seed=27)
    logits[0, 5], logits[1, 7] = -float("inf"), float("nan")
    ids = torch.tensor([[5, 1, 2], [3, 7, -1], [0, 4, -1], [9, 8, 7]], device=DEV)
    g = randn(4, 3, seed=28)
    clean = g.clone()
    clean[0, 0] = clean[1, 1] = clean[1, 2] = clean[2, 2] = 0
    g[0, 0], g[1, 1], g[1, 2], g[2, 2] = float("inf"), float("nan"), float("nan"), float("inf")
    got, want = (moe_ops.route_topk_backward(t, ids, logits, scoring=scoring, renormalize=renormalize) for t in (g, clean))
    assert bool(torch.isfinite(want).all()) and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(3, 200, 7168), (300, 520, 7168), (40, 96, 8192), (2100, 2080, 4096)])
def test_the_sign_that_the_gradient_of_relu_turns_on(m, n, k, dtype):
    """Long sums of one sign that the bias takes back to 1e-5 of themselves: z is positive everywhere, by more than what runs of 512
    terms lose (5.6e-6 of the sum: 40 steps of 2^-23 and one of 2^-24 for each of at most 16 runs) and less than what one run of all does."""
    x, w = randn(1, k, seed=29, dtype=dtype).abs().expand(m, k).contiguous(), randn(n, k, seed=30, dtype=dtype, scale=0.02).abs()
    sums = (x[:1].double() @ w.double().t()).view(-1)
    bias = (-sums * (1 - 1e-5)).float()
    z = sums + bias.double()
    assert bool((z > sums * 9.8e-6).all())
    y, pre = dense_ops.linear(x, w, bias=bias, activation="relu", return_pre=True)
    assert bool((pre > 0).all()) and bool((y > 0).all())
    assert bool(((pre.double() - z).abs() <= sums * 6e-6 + z * torch.finfo(dtype).eps).all())
    dy = torch.ones((m, n), dtype=dtype, device=DEV)
    db = dense_ops.linear_backward(dy, x, w, activation="relu", pre=pre, need_x=False, need_weight=False, bias_dtype=torch.float32)[2]
    assert bool((db == m).all())
    leaf = bias.clone().requires_grad_(True)
    assert bool((torch.autograd.grad(dense_ops.linear(x, w, bias=leaf, activation="relu").sum(), leaf)[0] == m).all())
