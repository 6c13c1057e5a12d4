"""Operators around the grouped GEMMs past 2^31 elements, with the same expert many times over, and called from several threads at once."""
import threading

import pytest
import torch

import asymgemm_b200 as ag
from asymgemm_b200 import dense_ops, moe_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def randn(*shape, seed=0, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)) * scale).to(dtype)


def tall(rows, cols, seed, dtype=torch.bfloat16):
    """Random rows in pieces, so that no temporary is as large as the tensor."""
    out = torch.empty((rows, cols), dtype=dtype, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for part in out.split(1 << 16):
        part.normal_(generator=gen)
    return out


def test_products_and_gradients_with_more_than_2_to_31_outputs():
    m, n, k = 270_000, 8192, 64
    x, w, b = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5), randn(n, seed=3)
    assert m * n > 1 << 31
    y, pre = dense_ops.linear(x, w, bias=b, activation="silu", return_pre=True)
    for rows in (slice(0, 300), slice(m // 2, m // 2 + 300), slice(m - 300, m)):
        part, part_pre = dense_ops.linear(x[rows], w, bias=b, activation="silu", return_pre=True)
        # the same sums of 64 terms, whatever tile they were computed in: half a step of bf16 twice, should one differ in its last bit
        for got, want in ((y[rows], part), (pre[rows], part_pre)):
            assert bool(((got.double() - want.double()).abs() <= want.double().abs() * 2 ** -7 + 2 ** -20).all())
    dy = y.zero_()      # no more memory than needed: a gradient that is 0 but for the last rows
    dy[m - 300:] = randn(300, n, seed=4)
    dx, dw, db = dense_ops.linear_backward(dy, x, w, activation="silu", pre=pre)
    part = dense_ops.linear_backward(dy[m - 300:], x[m - 300:], w, activation="silu", pre=pre[m - 300:], bias_dtype=torch.bfloat16)
    assert float(dx[: m - 300].abs().max()) == 0
    for got, want in ((dx[m - 300:], part[0]), (dw, part[1]), (db, part[2])):
        scale = float(want.double().abs().max())
        assert float((got.double() - want.double()).abs().max()) <= scale * 2 ** -7
    ag.check_status()


def test_router_and_its_gradient_past_2_to_31_logits():
    tokens, experts, k = 8_400_000, 256, 8
    logits = tall(tokens, experts, 5)
    assert logits.numel() > 1 << 31
    ids, w = moe_ops.route_topk(logits, k, renormalize=False)
    dw = randn(tokens, k, seed=6, dtype=torch.float32)
    dl = moe_ops.route_topk_backward(dw, ids, logits, renormalize=False)
    for rows in (slice(0, 700), slice(tokens // 2 + 1, tokens // 2 + 701), slice(tokens - 700, tokens)):
        part = moe_ops.route_topk(logits[rows], k, renormalize=False)
        assert torch.equal(ids[rows], part[0]) and torch.equal(w[rows], part[1])
        assert torch.equal(dl[rows], moe_ops.route_topk_backward(dw[rows], ids[rows], logits[rows], renormalize=False))


def test_combine_and_its_gradient_past_2_to_31_elements():
    tokens, k, cols = 66_000, 5, 7168
    rows = tall(tokens * k, cols, 7)
    assert rows.numel() > 1 << 31
    pos = torch.randperm(tokens * k, device=DEV, generator=torch.Generator(device=DEV).manual_seed(8))
    w, dy = torch.rand((tokens, k), device=DEV), randn(tokens, cols, seed=9)
    y = moe_ops.combine_topk(rows, pos, w, tokens, k)
    drows, dweights = moe_ops.combine_topk_backward(dy, rows, pos, w)
    for at in (slice(0, 50), slice(tokens - 50, tokens)):
        p = pos[at.start * k:at.stop * k]
        picked = rows[p]
        assert torch.equal(y[at], moe_ops.combine_topk(picked, None, w[at], 50, k))
        part = moe_ops.combine_topk_backward(dy[at], picked, None, w[at])
        assert torch.equal(drows[p], part[0]) and torch.equal(dweights[at], part[1])
    ag.check_status()


@pytest.mark.parametrize("tokens,experts,k", [(40, 5, 8), (900, 3, 7), (3000, 1, 4), (70000, 300, 8)])
def test_layouts_where_a_token_names_an_expert_more_than_once(tokens, experts, k):
    """More slots than experts, one expert for all: the same stable sort."""
    gen = torch.Generator().manual_seed(tokens)
    ids = torch.randint(0, experts, (tokens, k), generator=gen)
    if experts > 100:
        ids[:] = 131
    ids[::7, 1] = -1
    got = moe_ops.route_layout(ids.to(DEV), experts)
    flat = ids.view(-1)
    order = torch.argsort(torch.where(flat < 0, experts, flat), stable=True)[: int((flat >= 0).sum())]
    count = torch.bincount(flat[flat >= 0], minlength=experts)
    padded = (count + 127) // 128 * 128
    start = torch.cumsum(padded, 0) - padded
    within = torch.arange(order.numel()) - (torch.cumsum(count, 0) - count)[flat[order]]
    want = torch.full((tokens * k,), -1)
    want[order] = start[flat[order]] + within
    assert torch.equal(got.pair_row.cpu(), want) and torch.equal(got.rows_per_expert.cpu(), count)
    row_token = torch.full((got.row_token.numel(),), -1)
    row_token[want[order]] = order // k
    assert torch.equal(got.row_token.cpu(), row_token)
    room = max(1, int(count.max()) - 5)
    masked = moe_ops.route_layout_masked(ids.to(DEV), experts, room)
    fits = torch.where(within < room, flat[order] * room + within, -1)
    want[order] = fits
    assert torch.equal(masked.pair_row.cpu(), want) and torch.equal(masked.masked_m.cpu().long(), count.clamp(max=room))


def test_calls_from_several_threads_at_once():
    """Each thread on a stream of its own: products with workspaces, routing, layouts and gradients share nothing."""
    def step(seed):
        x, w = randn(900, 520, seed=seed), randn(264, 520, seed=seed + 1, scale=0.05)
        dy, pre = randn(900, 264, seed=seed + 2), randn(900, 264, seed=seed + 3)
        logits = randn(900, 96, seed=seed + 4, dtype=torch.float32)
        out = [dense_ops.linear(x, w, activation="gelu"), *dense_ops.linear_backward(dy, x, w, activation="gelu", pre=pre)]
        ids, weights = moe_ops.route_topk(logits, 4, scoring="sigmoid")
        lay = moe_ops.route_layout(ids, 96)
        rows = moe_ops.move_rows(dy, lay.row_token.numel(), src_rows=lay.row_token)
        y = moe_ops.combine_topk(rows, lay.pair_row, weights, 900, 4)
        return out + [ids, weights, lay.pair_row, y, *moe_ops.combine_topk_backward(pre, rows, lay.pair_row, weights)]

    want = [step(100 * i) for i in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(15):
                    got = step(100 * i)
                torch.cuda.current_stream().synchronize()
                wrong.extend((i, j) for j, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
        except Exception as e:
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
