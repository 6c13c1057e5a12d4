"""Routing to experts on the GPU: choice, weights and their gradient, the layout tables, the combine's gradient, and a run of
them together, against plain restatements in 64 bits."""
import math

import pytest
import torch

import asymgemm_b200 as ag
from asymgemm_b200 import moe_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
MAXF = torch.finfo(torch.float32).max


def clean(v):
    v = v.double()
    return torch.where(torch.isnan(v), -math.inf, v.clamp(max=MAXF))


def plain_route(logits, k, scoring, bias=None, groups=1, top_groups=1, group_score="top2", renormalize=True, scale=1.0, used=None):
    """Token by token in 64 bits."""
    logits = clean(logits.cpu())
    bias = None if bias is None else clean(bias.cpu())
    t, e = logits.shape
    ids = torch.full((t, k), -1, dtype=torch.int64)
    weights = torch.zeros((t, k), dtype=torch.float64)
    for i in range(t if used is None else used):
        l = logits[i]
        on = l > -math.inf
        if not bool(on.any()):
            continue
        s = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, 0)
        c = s if bias is None else s + bias
        if bias is not None:
            on = on & (bias > -math.inf)
        live = [x for x in range(e) if bool(on[x])]
        if groups > 1:
            size = e // groups
            best = []
            for g in range(groups):
                mine = sorted((float(c[x]) for x in live if x // size == g), reverse=True)
                best.append(((-math.inf if not mine else mine[0] if group_score == "max" else sum(mine[:2])), -g))
            keep = {-g for _, g in sorted(best, reverse=True)[:top_groups]}
            live = [x for x in live if x // size in keep]
        order = l if bias is None else c
        live.sort(key=lambda x: (-float(order[x]), x))
        picked = live[:k]
        if not picked:
            continue
        # scores up to a factor where they are renormalised: very small ones keep their ratios
        if renormalize:
            top = max(float(l[x]) for x in picked)
            if scoring == "sigmoid":
                top = min(top, 0.0)
                w = [math.exp(float(l[x]) - top) / (1 + math.exp(float(l[x]))) if float(l[x]) < 0 else 1 / (1 + math.exp(-float(l[x]))) for x in picked]
            else:
                w = [math.exp(float(l[x]) - top) for x in picked]
            w = [v / sum(w) for v in w]
        else:
            w = [float(s[x]) for x in picked]
        ids[i, :len(picked)] = torch.tensor(picked)
        weights[i, :len(picked)] = torch.tensor(w, dtype=torch.float64) * scale
    return ids, weights


def weight_bound(logits):
    """Relative: an exponential of a difference d is off by 2^-24 |d| + 2^-22 (argument, expf), sums of up to 37 steps by 37 * 2^-24,
    twice (numerator and denominator) with a division and the scale. Absolute: what underflows in fp32."""
    finite = clean(logits.cpu())
    finite = finite[finite > -1e30].clamp(max=1e30)
    spread = float((finite.max() - finite.min()).clamp(max=110)) if finite.numel() else 0.0
    return 2 * (spread * 2 ** -24 + 2 ** -22 + 37 * 2 ** -24) + 2 ** -22


def check_route(logits, k, **kw):
    used = kw.pop("used", None)
    rows_used = None if used is None else torch.tensor([used], dtype=torch.int32, device=DEV)
    ids, weights = moe_ops.route_topk(logits, k, rows_used=rows_used, **kw)
    names = dict(num_groups="groups", top_groups="top_groups")
    want_ids, want_w = plain_route(logits, k, kw.get("scoring", "softmax"), kw.get("bias"), kw.get("num_groups", 1), kw.get("top_groups", 1),
                                   kw.get("group_score", "top2"), kw.get("renormalize", True), kw.get("scale", 1.0), used)
    assert ids.dtype == torch.int64 and weights.dtype == torch.float32 and ids.shape == weights.shape == want_ids.shape, names
    assert torch.equal(ids.cpu(), want_ids)
    tol = weight_bound(logits)
    off = (weights.cpu().double() - want_w).abs()
    assert bool((off <= tol * want_w.abs() + 2 ** -120).all()), float((off / want_w.abs().clamp(min=1e-30)).max())
    return ids, weights


def randn(*shape, seed=0, dtype=torch.float32, scale=2.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (37, 32, 8), (9, 33, 32), (21, 60, 4), (7, 128, 6), (33, 256, 8),
                                              (6, 257, 9), (5, 512, 8), (4, 1000, 16), (3, 1024, 32)])
def test_choice_and_weights_without_groups(tokens, experts, k, dtype):
    logits = randn(tokens, experts, seed=experts, dtype=dtype)
    bias = randn(experts, seed=1, scale=0.05)
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            check_route(logits, k, scoring=scoring, renormalize=renormalize, scale=2.5)
            check_route(logits, k, scoring=scoring, renormalize=renormalize, bias=bias)


@pytest.mark.parametrize("experts,groups,top_groups,k", [(256, 8, 4, 8), (160, 8, 3, 6), (64, 2, 1, 5), (40, 5, 2, 4), (24, 8, 8, 24), (32, 32, 7, 7),
                                                         (1024, 8, 1, 32), (15, 3, 2, 4), (96, 32, 4, 12)])
def test_choice_within_groups(experts, groups, top_groups, k):
    logits = randn(29, experts, seed=experts + groups)
    bias = randn(experts, seed=3, scale=0.1)
    for scoring in ("softmax", "sigmoid"):
        for group_score in ("top2", "max"):
            for b in (None, bias):
                check_route(logits, k, scoring=scoring, bias=b, num_groups=groups, top_groups=top_groups, group_score=group_score, scale=1.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_equal_scores_go_to_the_lowest_index(scoring):
    for bias in (None, torch.zeros(64, device=DEV)):
        check_route(torch.zeros((3, 64), device=DEV), 6, scoring=scoring, bias=bias)
        check_route(torch.zeros((3, 64), device=DEV), 6, scoring=scoring, bias=bias, num_groups=4, top_groups=2)
        # a coarse grid of logits: many equal ones in every row
        check_route((randn(200, 64, seed=5) * 2).round() / 2, 6, scoring=scoring, bias=bias, num_groups=4, top_groups=2)
        check_route(randn(200, 64, seed=6, dtype=torch.bfloat16), 6, scoring=scoring, bias=bias)


def test_scores_that_fp32_cannot_tell_apart_are_ordered_as_in_64_bits():
    gen = torch.Generator().manual_seed(8)
    tokens, experts = 64, 128
    logits = torch.randn((tokens, experts), generator=gen)
    # biases that bring every expert of token 0 to the same choice, up to the rounding of the bias itself
    bias = (0.75 - torch.sigmoid(logits[0].double())).float()
    logits[1:] = logits[0] + (torch.rand((tokens - 1, experts), generator=gen) - 0.5) * 2e-6
    for groups, top in ((1, 1), (8, 3)):
        check_route(logits.to(DEV), 8, scoring="sigmoid", bias=bias.to(DEV), num_groups=groups, top_groups=top)
    soft = (0.75 - torch.softmax(logits[0].double(), 0)).float()
    check_route(logits.to(DEV), 8, scoring="softmax", bias=soft.to(DEV))
    # small scores that vanish beside each other in fp32
    check_route(torch.linspace(-60, 0, experts).repeat(4, 1).to(DEV), 8, scoring="softmax", bias=torch.zeros(experts, device=DEV))


@pytest.mark.parametrize("k", [1, 5, 8, 12])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 4)])
def test_two_experts_that_meet_at_the_border(k, groups, top_groups):
    """In every row the expert that is just chosen and the one that is just left out differ by 0 to a few hundred steps of fp32."""
    gen = torch.Generator().manual_seed(k + groups)
    tokens, experts = 640, 128
    logits = torch.randn((tokens, experts), generator=gen) * 1.5
    bias = torch.randn(experts, generator=gen) * 0.05
    step = torch.randint(-400, 401, (tokens,), generator=gen).double() * 2.0 ** -26 * torch.randint(0, 2, (tokens,), generator=gen)
    # among equals in the same groups: the reference's own order says which experts stand at the border
    order = plain_route(logits, k + 1, "sigmoid", bias, groups, top_groups)[0]
    at, out = order[:, k - 1], order[:, k]
    rows = torch.arange(tokens)
    choice = torch.sigmoid(logits[rows, at].double()) + bias[at].double() + step
    wanted = (choice - bias[out].double()).clamp(1e-3, 1 - 1e-3)
    logits[rows, out] = torch.log(wanted / (1 - wanted)).float()
    check_route(logits.to(DEV), k, scoring="sigmoid", bias=bias.to(DEV), num_groups=groups, top_groups=top_groups)
    # logits alone: neighbours in fp32, and equal ones
    order = plain_route(logits, k + 1, "softmax", None, groups, top_groups, "max")[0]
    at, out = order[:, k - 1], order[:, k]
    logits[rows, out] = torch.nextafter(logits[rows, at], torch.where(rows % 3 == 0, logits[rows, at], torch.where(rows % 3 == 1, 1e9, -1e9)))
    check_route(logits.to(DEV), k, num_groups=groups, top_groups=top_groups, group_score="max")
    check_route(logits.to(DEV), k, scoring="softmax", bias=torch.zeros(experts, device=DEV), num_groups=groups, top_groups=top_groups, group_score="max")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_experts_that_are_off_and_values_without_end(scoring):
    logits = randn(12, 48, seed=11)
    logits[0] = -math.inf                                   # no expert at all
    logits[1, :45] = -math.inf                              # fewer than top_k
    logits[2, ::3] = math.nan
    logits[3, 5] = math.inf
    logits[4, 5:9] = math.inf
    logits[5] = math.nan
    logits[6] = torch.finfo(torch.float32).min              # the type's lowest value is a finite logit
    logits[7] = -200 + torch.arange(48, device=DEV) * 0.1   # scores below the smallest fp32
    logits[8, 1:] = -math.inf
    bias = randn(48, seed=12, scale=0.1)
    bias[7] = -math.inf
    bias[9] = math.nan
    for b in (None, bias):
        for renormalize in (True, False):
            for groups, top in ((1, 1), (6, 2)):
                check_route(logits, 5, scoring=scoring, bias=b, renormalize=renormalize, num_groups=groups, top_groups=top)


def test_padding_tokens_strided_rows_and_empty_batches():
    wide = randn(40, 300, seed=13)
    view = wide[:, 7:7 + 256]
    for used in (0, 1, 25, 40):
        check_route(view, 8, scoring="sigmoid", num_groups=8, top_groups=4, used=used)
    check_route(wide[::3, :64], 4, used=9)
    ids, weights = moe_ops.route_topk(torch.empty((0, 64), device=DEV), 4)
    assert ids.shape == weights.shape == (0, 4)
    # another stream than the default one, and outputs of two calls at once
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = moe_ops.route_topk(view, 8)
    b = moe_ops.route_topk(view, 8)
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------------------------------ gradient
def plain_weights(logits, ids, scoring, renormalize, scale):
    """Differentiable weights of the chosen experts (ids >= 0), in 64 bits."""
    s = torch.sigmoid(logits) if scoring == "sigmoid" else torch.softmax(logits, 1)
    w = torch.where(ids >= 0, s.gather(1, ids.clamp(min=0)), 0)
    if renormalize:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    return w * scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (5, 7, 3), (33, 64, 8), (17, 60, 4), (9, 256, 8), (3, 1000, 32)])
def test_gradient_of_the_weights(tokens, experts, k, dtype):
    logits = randn(tokens, experts, seed=20 + experts, dtype=dtype, scale=1.5)
    g = randn(tokens, k, seed=21, scale=1.0)
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            used = max(1, tokens - 2)
            ids, weights = moe_ops.route_topk(logits, k, scoring=scoring, renormalize=renormalize, scale=1.5,
                                              rows_used=torch.tensor([used], dtype=torch.int32, device=DEV))
            got = moe_ops.route_topk_backward(g, ids, logits, scoring=scoring, renormalize=renormalize, scale=1.5)
            x = logits.cpu().double().requires_grad_(True)
            w = plain_weights(x, ids.cpu(), scoring, renormalize, 1.5)
            want, = torch.autograd.grad(w, x, torch.where(ids.cpu() >= 0, g.cpu().double(), 0))
            # every term is a product of a score (2^-18, see weight_bound: spread below 16) with a gradient and a sum of k such; the
            # largest of them bounds what cancellation leaves, then the result is rounded once to the type
            size = 2.5 * float(g.abs().max()) * 1.5
            tol = 2 ** -18 * size
            off = (got.cpu().double() - want).abs()
            assert got.dtype == dtype and bool((off <= tol + want.abs() * torch.finfo(dtype).eps / 2 + 2 ** -24 * (dtype == torch.float16)).all()), float(off.max())
            if dtype == torch.float32:
                leaf = logits.clone().requires_grad_(True)
                again, = torch.autograd.grad(moe_ops.route_topk(leaf, k, scoring=scoring, renormalize=renormalize, scale=1.5)[1], leaf, g)
                full = moe_ops.route_topk_backward(g, moe_ops.route_topk(logits, k, scoring=scoring)[0], logits, scoring=scoring, renormalize=renormalize, scale=1.5)
                assert torch.equal(again, full)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_against_differences(scoring, renormalize):
    logits = randn(4, 12, seed=30, scale=1.0)
    ids, _ = moe_ops.route_topk(logits, 3, scoring=scoring)
    g = randn(4, 3, seed=31, scale=1.0)
    got = moe_ops.route_topk_backward(g, ids, logits, scoring=scoring, renormalize=renormalize, scale=2.0).cpu().double()
    x, ids, g = logits.cpu().double(), ids.cpu(), g.cpu().double()
    step = 1e-5
    for e in range(12):
        d = torch.zeros_like(x)
        d[:, e] = step
        up, down = (plain_weights(x + s * d, ids, scoring, renormalize, 2.0) for s in (1, -1))
        num = ((up - down) * g).sum(1) / (2 * step)
        # central differences: third derivatives (below 8 here) times step^2 / 6, and 64-bit rounding over step
        assert torch.allclose(got[:, e], num, rtol=0, atol=1e-5), e


def test_gradient_of_named_twice_missing_and_switched_off_experts():
    logits = randn(5, 20, seed=33)
    logits[1, 4] = -math.inf
    logits[2] = math.nan
    ids = torch.tensor([[3, 3, 7], [4, 2, -1], [0, 1, 2], [25, -7, 6], [-1, -1, -1]], device=DEV)
    g = randn(5, 3, seed=34, scale=1.0)
    got = moe_ops.route_topk_backward(g, ids, logits, scoring="sigmoid", renormalize=False).cpu().double()
    s = torch.sigmoid(logits.cpu().double())
    want = torch.zeros(5, 20, dtype=torch.float64)
    for t, slots in enumerate(ids.cpu().tolist()):
        for j, e in enumerate(slots):
            if 0 <= e < 20 and bool(torch.isfinite(logits[t, e])):
                want[t, e] += float(g[t, j]) * float(s[t, e] * (1 - s[t, e]))
    assert torch.allclose(got, want, rtol=2 ** -20, atol=2 ** -22)
    soft = moe_ops.route_topk_backward(g, ids, logits, scoring="softmax", renormalize=False)
    assert bool(torch.isfinite(soft).all()) and float(soft[2].abs().max()) == 0 and float(soft[1, 4]) == 0 and float(soft[4].abs().max()) == 0
    assert moe_ops.route_topk_backward(g[:0], ids[:0], logits[:0]).shape == (0, 20)


# ------------------------------------------------------------------------------------------------------ layouts
def plain_layout(ids, experts, rows, alignment=128, max_rows=0):
    flat = ids.cpu().reshape(-1).tolist()
    k = ids.shape[1]
    lists = [[i for i, e in enumerate(flat) if e == x] for x in range(experts)]
    pair_row = torch.full((len(flat),), -1, dtype=torch.int64)
    row_token = torch.full((rows,), -1, dtype=torch.int64)
    start, offsets = 0, []
    for x, pairs in enumerate(lists):
        if max_rows:
            start, pairs = x * max_rows, pairs[:max_rows]
        for n, i in enumerate(pairs):
            pair_row[i] = start + n
            row_token[start + n] = i // k
        end = start + -(-len(pairs) // alignment) * alignment
        offsets += [start, end]
        start = end
    return pair_row, row_token, torch.tensor([len(v) for v in lists]), torch.tensor(offsets, dtype=torch.int32), lists


def make_ids(tokens, experts, k, seed, missing=0.0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.rand((tokens, experts), generator=gen).mul_(torch.rand(experts, generator=gen)).topk(k, dim=1).indices
    if missing:
        ids[torch.rand(ids.shape, generator=gen) < missing] = -1
    return ids


@pytest.mark.parametrize("tokens,experts,k", [(0, 4, 2), (1, 1, 1), (1, 256, 8), (5, 3, 2), (64, 256, 8), (512, 8, 8), (513, 8, 8), (1365, 60, 3),
                                              (3000, 16, 4), (9000, 256, 8), (700, 1024, 7), (40000, 5, 1)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_contiguous_layout(tokens, experts, k, dtype):
    for missing, alignment in ((0.0, 128), (0.3, 128), (0.1, 1)):
        ids = make_ids(tokens, experts, k, tokens + experts, missing).to(dtype).to(DEV)
        got = moe_ops.route_layout(ids, experts, alignment)
        rows = got.row_token.numel()
        pair_row, row_token, count, offsets, _ = plain_layout(ids, experts, rows, alignment)
        assert torch.equal(got.pair_row.cpu(), pair_row) and torch.equal(got.row_token.cpu(), row_token)
        assert torch.equal(got.rows_per_expert.cpu(), count) and torch.equal(got.offsets.cpu(), offsets)
        assert got.experts.tolist() == list(range(experts)) + [-1] and got.experts.dtype == torch.int32


@pytest.mark.parametrize("tokens,experts,k", [(256, 256, 8), (2048, 16, 1), (2049, 16, 1), (150001, 7, 4), (131073, 60, 4), (700000, 3, 1)])
def test_layouts_on_either_side_of_their_block_sizes(tokens, experts, k):
    """One block, several, and so many pairs that a block's do not stay in registers; every table of both layouts."""
    ids = make_ids(tokens, experts, k, tokens + experts, 0.1).to(DEV)
    got = moe_ops.route_layout(ids, experts)
    pair_row, row_token, count, offsets, _ = plain_layout(ids, experts, got.row_token.numel())
    assert torch.equal(got.pair_row.cpu(), pair_row) and torch.equal(got.row_token.cpu(), row_token)
    assert torch.equal(got.rows_per_expert.cpu(), count) and torch.equal(got.offsets.cpu(), offsets)
    max_rows = tokens * k // experts
    masked = moe_ops.route_layout_masked(ids, experts, max_rows)
    # the same order within an expert, its rows elsewhere and no more than max_rows of them
    flat = ids.view(-1).cpu()
    within = pair_row - offsets.view(-1, 2)[flat.clamp(min=0), 0]
    want = torch.where((flat >= 0) & (within < max_rows), flat * max_rows + within, -1)
    assert torch.equal(masked.pair_row.cpu(), want) and torch.equal(masked.masked_m.cpu().long(), count.clamp(max=max_rows))
    tokens_of = torch.full((experts * max_rows,), -1, dtype=torch.int64)
    tokens_of[want[want >= 0]] = (torch.arange(tokens * k) // k)[want >= 0]
    assert torch.equal(masked.row_token.cpu(), tokens_of)


@pytest.mark.parametrize("tokens,experts,k,max_rows", [(0, 3, 2, 4), (1, 8, 2, 1), (64, 256, 8, 16), (100, 8, 4, 30), (4000, 16, 4, 600), (2000, 4, 2, 1500)])
def test_masked_layout_drops_what_does_not_fit(tokens, experts, k, max_rows):
    for missing in (0.0, 0.2):
        ids = make_ids(tokens, experts, k, tokens, missing).to(DEV)
        got = moe_ops.route_layout_masked(ids, experts, max_rows)
        pair_row, row_token, _, _, lists = plain_layout(ids, experts, experts * max_rows, max_rows=max_rows)
        assert torch.equal(got.pair_row.cpu(), pair_row) and torch.equal(got.row_token.cpu(), row_token)
        assert got.masked_m.tolist() == [min(len(v), max_rows) for v in lists] and got.masked_m.dtype == torch.int32


@pytest.mark.expects_status
def test_ids_outside_the_experts_are_left_out_and_reported():
    ids = make_ids(600, 16, 8, 5).to(DEV)
    ids[3, 2], ids[500, 7] = 16, -2
    got = moe_ops.route_layout(ids, 16)
    clean_ids = torch.where((ids < 0) | (ids >= 16), -1, ids)
    pair_row, row_token, count, offsets, _ = plain_layout(clean_ids, 16, got.row_token.numel())
    assert torch.equal(got.pair_row.cpu(), pair_row) and torch.equal(got.row_token.cpu(), row_token) and torch.equal(got.offsets.cpu(), offsets)
    with pytest.raises(RuntimeError, match="expert id"):
        ag.check_status()
    ag.check_status()


# ------------------------------------------------------------------------------------------------------ combine
def combine_case(tokens, experts, k, cols, dtype, seed, missing=0.2):
    ids = make_ids(tokens, experts, k, seed, missing).to(DEV)
    lay = moe_ops.route_layout(ids, experts)
    rows = randn(max(1, lay.row_token.numel()), cols, seed=seed, dtype=dtype, scale=1.0)
    weights = torch.softmax(randn(tokens, k, seed=seed + 1, scale=1.0), 1)
    dy = randn(tokens, cols, seed=seed + 2, dtype=torch.bfloat16, scale=1.0)
    return lay, rows, weights, dy


@pytest.mark.parametrize("tokens,experts,k,cols", [(1, 4, 1, 8), (3, 4, 2, 128), (50, 8, 4, 1024), (37, 60, 9, 1032), (20, 32, 17, 7168), (0, 4, 2, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_of_the_combine(tokens, experts, k, cols, dtype):
    lay, rows, weights, dy = combine_case(tokens, experts, k, cols, dtype, tokens + k)
    pos = lay.pair_row.cpu()
    live = (pos >= 0).view(tokens, k)
    picked = rows.cpu().double()[pos.clamp(min=0)].view(tokens, k, cols)
    w, g = weights.cpu().double(), dy.cpu().double()
    y = moe_ops.combine_topk(rows, lay.pair_row, weights, tokens, k).cpu().double()
    terms = torch.where(live.unsqueeze(2), picked * w.unsqueeze(2), 0)
    # k fused multiply-adds in fp32, one rounding to bf16
    assert bool(((y - terms.sum(1)).abs() <= terms.abs().sum(1) * k * 2 ** -24 + terms.sum(1).abs() * 2 ** -8).all())

    drows, dweights = moe_ops.combine_topk_backward(dy, rows, lay.pair_row, weights)
    products = torch.where(live.unsqueeze(2), picked * g.unsqueeze(1), 0)
    # a thread adds cols / 128 products (8 columns at a time), then 5 + 4 joining steps
    steps = cols / 128 + 8 + 9
    assert bool(((dweights.cpu().double() - products.sum(2)).abs() <= products.abs().sum(2) * steps * 2 ** -24).all())
    want = torch.zeros(rows.shape, dtype=torch.float64)
    sel = live.view(-1).nonzero().view(-1)
    want[pos[sel]] = (w.unsqueeze(2) * g.unsqueeze(1)).view(-1, cols)[sel]
    eps = torch.finfo(dtype).eps / 2 + 2 ** -24
    assert drows.dtype == dtype and bool(((drows.cpu().double() - want).abs() <= want.abs() * eps).all())

    none, only = moe_ops.combine_topk_backward(dy, rows, lay.pair_row, weights, need_rows=False)
    assert none is None and torch.equal(only, dweights)
    only, none = moe_ops.combine_topk_backward(dy, rows, lay.pair_row, weights, need_weights=False)
    assert none is None and torch.equal(only, drows)
    a, b = rows.clone().requires_grad_(True), weights.clone().requires_grad_(True)
    got = torch.autograd.grad(moe_ops.combine_topk(a, lay.pair_row, b, tokens, k), (a, b), dy)
    assert torch.equal(got[0], drows) and torch.equal(got[1], dweights)


def test_gradient_of_the_combine_where_plain_torch_computes_it():
    """Types and widths without a kernel: float16, and bf16 rows of 12 columns."""
    for dtype, cols in ((torch.float16, 64), (torch.bfloat16, 12)):
        lay, rows, weights, _ = combine_case(9, 4, 2, cols, dtype, 33)
        a, b = rows.clone().requires_grad_(True), weights.clone().requires_grad_(True)
        y = moe_ops.combine_topk(a, lay.pair_row, b, 9, 2)
        dy = randn(9, cols, seed=34, dtype=dtype, scale=1.0)
        drows, dweights = torch.autograd.grad(y, (a, b), dy)
        pos = lay.pair_row.cpu()
        live = pos >= 0
        g, w = dy.cpu().double().repeat_interleave(2, 0), weights.cpu().double().view(-1, 1)
        want = torch.zeros(rows.shape, dtype=torch.float64)
        want[pos[live]] = (w * g)[live]
        assert bool(((drows.cpu().double() - want).abs() <= want.abs() * (torch.finfo(dtype).eps / 2 + 2 ** -23)).all())
        terms = torch.where(live.view(-1, 1), rows.cpu().double()[pos.clamp(min=0)] * g, 0)
        # a product and at most `cols` additions in fp32
        assert bool(((dweights.cpu().double().view(-1) - terms.sum(1)).abs() <= terms.abs().sum(1) * (cols + 1) * 2 ** -24).all())


def test_position_tables_may_be_longer_than_the_batch():
    lay, rows, weights, dy = combine_case(11, 4, 2, 64, torch.bfloat16, 35)
    longer = torch.cat([lay.pair_row, torch.full((9,), 5, device=DEV)])
    grads = []
    for pos in (lay.pair_row, longer):
        a, b = rows.clone().requires_grad_(True), weights.clone().requires_grad_(True)
        grads.append(torch.autograd.grad(moe_ops.combine_topk(a, pos, b, 11, 2), (a, b), dy))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


def test_layers_record_no_gradient():
    """The layers' GEMMs have no gradient, so their output claims none either, whatever the weights ask for."""
    from asymgemm_b200.ep import EPDispatcher
    disp = EPDispatcher(8)
    ids, x, w = make_ids(20, 8, 2, 36).to(DEV), randn(20, 64, seed=37, dtype=torch.bfloat16), torch.rand((20, 2), device=DEV, requires_grad=True)
    state, _, _ = disp.dispatch(x, ids)
    out = randn(state.padded_rows, 64, seed=38, dtype=torch.bfloat16)
    assert not disp.combine(out, state, w).requires_grad
    assert moe_ops.combine_topk(out, state.tables.pair_row, w, 20, 2).requires_grad


@pytest.mark.expects_status
@pytest.mark.parametrize("tokens,k,cols,rows", [(1024, 4, 8, 5000), (1025, 4, 8, 5000), (3, 2, 8, 4194304), (3, 2, 8, 4194305), (700, 5, 8, 40001), (0, 3, 16, 77),
                                                (16, 2, 16384, 2048), (16, 2, 16384, 2049)])
def test_gradient_rows_with_and_without_flags(tokens, k, cols, rows):
    """Both sides of the sizes at which the rows that no pair names are found another way, and a row named twice in each."""
    gen = torch.Generator().manual_seed(rows)
    pos = torch.randint(rows, (4 * tokens * k,), generator=gen).unique()
    pos = pos[torch.randperm(pos.numel(), generator=gen)][: tokens * k]
    if tokens:
        pos[0], pos[1], pos[2] = rows, -1, rows - 1
        pos[3:] = torch.where(pos[3:] == rows - 1, -7, pos[3:])
    assert pos.numel() == tokens * k
    x, w = torch.randn((rows, cols), device=DEV).to(torch.bfloat16), torch.rand((tokens, k), device=DEV)
    dy = randn(tokens, cols, seed=39, dtype=torch.bfloat16, scale=1.0)
    drows, dweights = moe_ops.combine_topk_backward(dy, x, pos.to(DEV), w)
    live = ((pos >= 0) & (pos < rows)).to(DEV)
    at = pos.to(DEV)[live]
    want = torch.zeros((rows, cols), dtype=torch.float64, device=DEV)
    want[at] = (w.double().view(-1, 1) * dy.double().repeat_interleave(k, 0))[live]
    assert bool(((drows.double() - want).abs() <= want.abs() * (2 ** -8 + 2 ** -23)).all())
    terms = torch.zeros((tokens * k, cols), dtype=torch.float64, device=DEV)
    terms[live] = dy.double().repeat_interleave(k, 0)[live] * x[at].double()
    steps = cols / 128 + 8 + 9      # as above
    assert bool(((dweights.double().view(-1) - terms.sum(1)).abs() <= terms.abs().sum(1) * steps * 2 ** -24).all())
    ag.check_status()
    if tokens:
        pos[-1] = rows - 1
        moe_ops.combine_topk_backward(dy, x, pos.to(DEV), w)
        with pytest.raises(RuntimeError, match="same row"):
            ag.check_status()


def test_gradient_of_the_combine_without_a_position_table():
    rows, w = randn(60, 256, seed=40, dtype=torch.bfloat16), torch.rand((20, 3), device=DEV)
    dy = randn(20, 256, seed=41, dtype=torch.bfloat16)
    drows, dweights = moe_ops.combine_topk_backward(dy, rows, None, w)
    pos = torch.arange(60, device=DEV)
    again = moe_ops.combine_topk_backward(dy, rows, pos, w)
    assert torch.equal(drows, again[0]) and torch.equal(dweights, again[1])


@pytest.mark.expects_status
def test_a_row_named_twice_is_reported_and_rows_outside_add_nothing():
    rows, w = randn(8, 64, seed=42, dtype=torch.bfloat16), torch.rand((4, 2), device=DEV)
    dy = randn(4, 64, seed=43, dtype=torch.bfloat16)
    pos = torch.tensor([0, 1, 2, 9, 4, -5, 6, 7], device=DEV)
    drows, dweights = moe_ops.combine_topk_backward(dy, rows, pos, w)
    ag.check_status()
    assert float(dweights[1, 1]) == 0 and float(dweights[2, 1]) == 0 and float(drows[3].abs().max()) == float(drows[5].abs().max()) == 0
    pos = torch.tensor([0, 1, 2, 3, 4, 3, 6, 7], device=DEV)
    moe_ops.combine_topk_backward(dy, rows, pos, w, need_rows=False)       # the weights' gradient has no such limit
    ag.check_status()
    moe_ops.combine_topk_backward(dy, rows, pos, w)
    with pytest.raises(RuntimeError, match="same row"):
        ag.check_status()


def test_row_moves_skip_missing_rows():
    src = randn(6, 32, seed=44)
    out = moe_ops.move_rows(src, 5, src_rows=torch.tensor([3, -1, 0, 5, -1], device=DEV))
    assert torch.equal(out[0], src[3]) and torch.equal(out[3], src[5]) and float(out[1].abs().max()) == float(out[4].abs().max()) == 0
    out = moe_ops.move_rows(src, 4, dst_rows=torch.tensor([2, -1, 0, -1, 3, -1], device=DEV), zero=True)
    assert torch.equal(out[2], src[0]) and torch.equal(out[0], src[2]) and torch.equal(out[3], src[4]) and float(out[1].abs().max()) == 0


# ------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    x = randn(4, 64, seed=50)
    for bad in (dict(top_k=0), dict(top_k=33), dict(top_k=65), dict(top_k=4, scoring="tanh"), dict(top_k=4, num_groups=5), dict(top_k=4, num_groups=0),
                dict(top_k=4, num_groups=8, top_groups=9), dict(top_k=17, num_groups=4, top_groups=1), dict(top_k=4, group_score="mean"),
                dict(top_k=4, bias=torch.zeros(63, device=DEV)), dict(top_k=4, bias=torch.zeros(64, device=DEV, dtype=torch.bfloat16)),
                dict(top_k=4, bias=torch.zeros(64)), dict(top_k=4, rows_used=torch.zeros(1, device=DEV)), dict(top_k=4, num_groups=64)):
        with pytest.raises(RuntimeError):
            moe_ops.route_topk(x, **bad)
    for bad in (x.cpu(), x[0], x.t(), x.double(), randn(2, 1025)):
        with pytest.raises(RuntimeError):
            moe_ops.route_topk(bad, 2)
    ids, w = moe_ops.route_topk(x, 4)
    for args in ((w[:, :3], ids, x), (w, ids[:3], x), (w.double(), ids, x), (w, ids.int(), x), (w.cpu(), ids, x)):
        with pytest.raises(RuntimeError):
            moe_ops.route_topk_backward(*args)
    for args in ((ids.float(), 64), (ids[0], 64), (ids, 0), (ids, 1025), (ids.cpu(), 64), (ids[:, ::2], 64), (ids, 64, 0)):
        with pytest.raises(RuntimeError):
            moe_ops.route_layout(*args)
    for rows in (0, -1, 1 << 30):
        with pytest.raises(RuntimeError):
            moe_ops.route_layout_masked(ids, 64, rows)
    rows, dy = randn(16, 64, dtype=torch.bfloat16), randn(4, 64, dtype=torch.bfloat16)
    pos = torch.arange(16, device=DEV)
    for args in ((dy.float(), rows, pos, w), (dy, rows[:, :32], pos, w), (dy, rows.half(), pos, w), (dy, rows, pos[:15], w), (dy, rows, pos.int(), w),
                 (dy[:3], rows, pos, w), (randn(4, 60, dtype=torch.bfloat16), randn(16, 60, dtype=torch.bfloat16), pos, w)):
        with pytest.raises(RuntimeError):
            moe_ops.combine_topk_backward(*args)


# ------------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("tokens,k", [(300, 4), (3000, 9)])
def test_route_layout_and_combine_together_in_a_captured_graph(tokens, k):
    """Logits -> ids, weights -> layout -> rows gathered, scaled by expert (in place of the experts' products) -> combine, and
    the way back to the logits, replayed on new inputs."""
    experts, cols, live = 24, 256, tokens - 20
    x, logits = randn(tokens, cols, seed=60, dtype=torch.bfloat16, scale=1.0), randn(tokens, experts, seed=61)
    used = torch.tensor([live], dtype=torch.int32, device=DEV)
    dy = randn(tokens, cols, seed=62, dtype=torch.bfloat16, scale=1.0)

    def step():
        ids, w = moe_ops.route_topk(logits, k, scoring="sigmoid", num_groups=4, top_groups=2, rows_used=used)
        lay = moe_ops.route_layout(ids, experts)
        a = moe_ops.move_rows(x, lay.row_token.numel(), src_rows=lay.row_token)
        y = moe_ops.combine_topk(a, lay.pair_row, w, tokens, k)
        _, dw = moe_ops.combine_topk_backward(dy, a, lay.pair_row, w, need_rows=False)
        return ids, w, y, moe_ops.route_topk_backward(dw, ids, logits, scoring="sigmoid")

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (70, 71):
        logits.copy_(randn(tokens, experts, seed=seed))
        x.copy_(randn(tokens, cols, seed=seed + 5, dtype=torch.bfloat16, scale=1.0))
        graph.replay()
        want = step()
        for got, w in zip(out, want):
            assert torch.equal(got, w)
    # every token's rows are its own x: the combine gives x back where the weights sum to 1
    y, xs = out[2][:live].double(), x[:live].double()
    assert bool(((y - xs).abs() <= xs.abs() * (2 ** -8 + 16 * 2 ** -22)).all()) and float(out[2][live:].abs().max()) == 0


@pytest.mark.parametrize("tokens,experts,k,cols,dtype", [(37, 8, 3, 64, torch.bfloat16), (1, 256, 8, 32, torch.bfloat16), (700, 60, 4, 20, torch.float32)])
def test_dispatcher_on_one_gpu_lays_rows_out_as_on_the_cpu(tokens, experts, k, cols, dtype):
    from asymgemm_b200.ep import EPDispatcher, to_contiguous_layout
    disp = EPDispatcher(experts)
    ids, x = make_ids(tokens, experts, k, 90), randn(tokens, cols, seed=91, dtype=dtype)
    w = torch.rand((tokens, k), generator=torch.Generator().manual_seed(92))
    cpu, rows_cpu, _ = disp.dispatch(x.cpu(), ids)
    gpu, rows_gpu, _ = disp.dispatch(x, ids.to(DEV))
    a_cpu, a_gpu = to_contiguous_layout(rows_cpu, cpu), to_contiguous_layout(rows_gpu, gpu)
    assert torch.equal(a_gpu.cpu(), a_cpu) and gpu.padded_rows == cpu.padded_rows
    assert torch.equal(gpu.offsets.cpu(), cpu.offsets) and torch.equal(gpu.experts.cpu(), cpu.experts)
    assert torch.equal(gpu.rows_per_expert.cpu(), cpu.rows_per_expert)
    y_cpu, y_gpu = disp.combine(a_cpu, cpu, w), disp.combine(a_gpu, gpu, w.to(DEV))
    # k products and additions in fp32, then one rounding to bf16 (the CPU rounds to the rows' type)
    size = (a_cpu.double().abs().max() * w.double().sum(1).max()).item()
    assert bool(((y_gpu.cpu().double() - y_cpu.double()).abs() <= 2 ** -7 * y_cpu.double().abs() + size * 2 * k * 2 ** -24).all())
