"""The router over batches large enough for several tokens per warp (top_k up to 8), where rows of all kinds meet in one warp: against
the definition in 64 bits, over whole batches at once."""
import math

import pytest
import torch

from asymgemm_b200 import moe_ops
from tests.test_gpu_route import clean, weight_bound

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain(logits, k, scoring, bias, groups, top_groups, group_score, renormalize, scale, used):
    l = clean(logits)
    t, e = l.shape
    on = l > -math.inf
    s = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(torch.where(on.any(1, keepdim=True), l, 0), 1)
    c = s if bias is None else s + clean(bias)
    order = torch.where(on, l if bias is None else c, -math.inf)
    if groups > 1:
        best = torch.where(on, c, -math.inf).view(t, groups, e // groups).sort(dim=2, descending=True).values
        two = best[:, :, :1].sum(2) if group_score == "max" or e == groups else torch.where(best[:, :, 1] == -math.inf, best[:, :, 0], best[:, :, 0] + best[:, :, 1])
        keep = two.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        kept = torch.zeros((t, groups), dtype=torch.bool, device=l.device).scatter_(1, keep, True)
        order = torch.where(kept.repeat_interleave(e // groups, 1), order, -math.inf)
    values, ids = order.sort(dim=1, descending=True, stable=True)
    ids, live = ids[:, :k], values[:, :k] > -math.inf
    live = live & (torch.arange(t, device=l.device) < used).unsqueeze(1)
    w = torch.where(live, s.gather(1, ids), 0)
    if renormalize:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    return torch.where(live, ids, -1), w * scale


def make(tokens, experts, dtype, seed, special):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn((tokens, experts), generator=gen) * 1.5).to(dtype)
    if special:      # one row in five is out of the ordinary, next to ordinary ones in its warp
        kind = torch.randint(0, 25, (tokens,), generator=gen)
        logits[kind == 0] = math.nan
        logits[kind == 1] = -math.inf
        logits[(kind == 2).nonzero(), ::3] = math.nan
        logits[(kind == 3).nonzero(), 2:] = -math.inf                # fewer than top_k
        logits[(kind == 4).nonzero(), experts // 2] = math.inf
        logits[(kind == 5).nonzero(), :: max(1, experts // 7)] = math.inf
        logits[kind == 6] = 0.25                                     # all equal
    return logits.to(DEV)


def check(logits, k, used=None, scoring="softmax", bias=None, groups=1, top_groups=1, group_score="top2", renormalize=True, scale=1.0):
    rows_used = None if used is None else torch.tensor([used], dtype=torch.int32, device=DEV)
    ids, weights = moe_ops.route_topk(logits, k, scoring=scoring, bias=bias, num_groups=groups, top_groups=top_groups, group_score=group_score,
                                      renormalize=renormalize, scale=scale, rows_used=rows_used)
    want_ids, want = plain(logits, k, scoring, bias, groups, top_groups, group_score, renormalize, scale, logits.shape[0] if used is None else used)
    wrong = (ids != want_ids).any(1).nonzero().view(-1)
    assert wrong.numel() == 0, (wrong[:5].tolist(), ids[wrong[:3]].tolist(), want_ids[wrong[:3]].tolist())
    off = (weights.double() - want).abs()
    assert bool((off <= weight_bound(logits) * want.abs() + 2 ** -120).all()), float((off / want.abs().clamp(min=1e-30)).max())


def biases(experts, seed):
    b = torch.randn(experts, generator=torch.Generator().manual_seed(seed)) * 0.05
    if experts > 20:
        b[3], b[11] = -math.inf, math.nan      # two experts that are off for every token
    return b.to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,experts", [(593, 8), (601, 60), (1203, 256), (602, 257), (1000, 128), (701, 1000), (600, 1024)])
def test_many_tokens_without_groups(tokens, experts, dtype):
    for special in (False, True):
        logits = make(tokens, experts, dtype, experts + special, special)
        for k in (1, 6, 8):
            for scoring in ("softmax", "sigmoid"):
                for renormalize in (True, False):
                    check(logits, k, tokens - 7, scoring, None, renormalize=renormalize, scale=2.5)
                    check(logits, k, None, scoring, biases(experts, 1), renormalize=renormalize)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts,groups,top_groups,k", [(1203, 256, 8, 4, 8), (601, 255, 3, 2, 8), (605, 60, 5, 2, 6), (999, 256, 16, 4, 8), (601, 64, 32, 9, 7),
                                                                (700, 1000, 8, 3, 8), (650, 24, 6, 1, 4), (603, 12, 12, 5, 5), (600, 512, 2, 1, 8)])
def test_many_tokens_within_groups(tokens, experts, groups, top_groups, k, dtype):
    for special in (False, True):
        logits = make(tokens, experts, dtype, experts + groups + special, special)
        for scoring in ("softmax", "sigmoid"):
            for group_score in ("top2", "max"):
                for bias in (None, biases(experts, 2)):
                    check(logits, k, tokens - 5, scoring, bias, groups, top_groups, group_score, renormalize=special, scale=1.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_tokens_in_strided_rows_and_padded_batches(dtype):
    wide = make(1300, 320, dtype, 9, True)
    bias = biases(256, 3)
    for rows in (wide[:, 5:261], wide[:, 32:288], wide[::2, 32:288]):      # unaligned, aligned, every other row
        for used in (0, 1, 599, 601, 602, 603, rows.shape[0], rows.shape[0] + 9):
            check(rows, 8, min(used, rows.shape[0]), "sigmoid", bias, 8, 4, scale=2.5)
            check(rows, 8, min(used, rows.shape[0]), "softmax", None, renormalize=False)


def test_the_two_sides_of_the_batch_size_agree():
    """592 tokens (4 per SM) take a row per warp, 593 several: the same rows, the same answer."""
    for experts, groups, top, k in ((256, 8, 4, 8), (60, 1, 1, 4), (250, 5, 2, 8)):
        logits, bias = make(700, experts, torch.float32, 31, True), biases(experts, 4)
        ids, w = moe_ops.route_topk(logits, k, scoring="sigmoid", bias=bias, num_groups=groups, top_groups=top)
        few = [moe_ops.route_topk(part, k, scoring="sigmoid", bias=bias, num_groups=groups, top_groups=top) for part in logits.split(100)]
        assert torch.equal(ids, torch.cat([a for a, _ in few]))
        assert bool(((w - torch.cat([b for _, b in few])).abs() <= 2 ** -20 * w.abs()).all())


def test_the_way_through_64_bits_for_many_rows_of_a_warp():
    """Equal scores in every row (a gate before training, sigmoids that are saturated) and equal ones at the border in some."""
    bias = torch.zeros(256, device=DEV)
    flat = torch.zeros((640, 256), device=DEV)
    for groups, top in ((1, 1), (8, 4)):
        check(flat, 8, None, "sigmoid", bias, groups, top)
        check(flat, 8, None, "softmax", bias, groups, top)
        check(flat, 8, None, "softmax", None, groups, top)
        check(flat + 40, 8, None, "sigmoid", bias, groups, top)
    mixed = make(1201, 256, torch.float32, 33, True)
    mixed[::3, 40:90] = 3.0
    mixed[1::5, 10:200] = 30.0 + torch.arange(190, device=DEV) * 0.01       # saturated: scores that fp32 cannot tell apart
    for groups, top in ((1, 1), (8, 4)):
        for scoring in ("sigmoid", "softmax"):
            check(mixed, 8, 1190, scoring, bias, groups, top)
            check(mixed, 5, None, scoring, biases(256, 6), groups, top)


@pytest.mark.parametrize("tokens,experts,groups,top_groups,k", [(5000, 256, 1, 1, 16), (5001, 256, 8, 4, 9), (4800, 60, 1, 1, 32), (2500, 1000, 8, 3, 12), (3001, 512, 16, 16, 20)])
def test_many_tokens_with_more_than_eight_experts_each(tokens, experts, groups, top_groups, k):
    """A row per warp, and several rows for each warp of the launch one after the other."""
    for dtype in (torch.float32, torch.bfloat16):
        logits = make(tokens, experts, dtype, experts + k, True)
        for scoring in ("softmax", "sigmoid"):
            for bias in (None, biases(experts, 7)):
                check(logits, k, tokens - 11, scoring, bias, groups, top_groups, renormalize=bias is None, scale=1.5)
