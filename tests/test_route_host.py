"""Routing, layout tables, combine gradient and dense product: what is refused, before anything is launched, and the CPU branches of
the row moves. No GPU is needed: pointers below are never dereferenced, every call returns from its checks."""
import ctypes

import pytest
import torch

from asymgemm_b200 import _lib, dense_ops, moe_ops

P = 0x7F0000000000      # a 256-byte aligned address
BAD, OK = _lib.AG_E_INVALID, _lib.AG_OK


def route_desc(**kw):
    d = _lib.RouteDesc()
    base = dict(logits=P, ld=64, ids=P, weights=P, tokens=4, dtype=2, experts=64, top_k=4, groups=1, top_groups=1, scoring=0, renormalize=1, scale=1.0)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


def test_router_refuses_bad_descriptors():
    lib = _lib.load()
    assert lib.ag_route_topk(None) == BAD
    for bad in (dict(dtype=3), dict(dtype=-1), dict(tokens=-1), dict(experts=0), dict(top_k=0), dict(top_k=33), dict(top_k=65), dict(ld=63), dict(scoring=2),
                dict(groups=0), dict(groups=3), dict(groups=33, experts=66, ld=66), dict(groups=8, top_groups=0), dict(groups=8, top_groups=9),
                dict(groups=8, top_groups=1, top_k=9), dict(experts=1056, ld=1056), dict(experts=2048, ld=2048, groups=32, top_groups=32),
                dict(experts=1000, ld=1000, groups=10, top_groups=4), dict(logits=P + 2), dict(ids=P + 4), dict(weights=P + 2), dict(bias=P + 1),
                dict(rows_used=P + 2), dict(logits=None), dict(ids=None), dict(weights=None), dict(tokens=1 << 40)):
        assert lib.ag_route_topk(route_desc(**bad)) == BAD, bad
        assert _lib.last_error()
    assert lib.ag_route_topk(route_desc(tokens=0, logits=None)) == OK
    assert lib.ag_route_topk(route_desc(tokens=0, dtype=0, logits=P + 2)) == OK

    def back(logits=P, dtype=2, tokens=4, ld=64, experts=64, dw=P, ids=P, k=4, scoring=0, out=P):
        return lib.ag_route_topk_backward(logits, dtype, tokens, ld, experts, dw, ids, k, scoring, 1, 1.0, out, None)

    for bad in (dict(dtype=5), dict(tokens=-1), dict(ld=60), dict(experts=0), dict(k=0), dict(k=33), dict(scoring=-1), dict(logits=P + 1), dict(out=P + 2),
                dict(dw=P + 2), dict(ids=P + 4), dict(logits=None), dict(dw=None), dict(ids=None), dict(out=None)):
        assert back(**bad) == BAD, bad
    assert back(tokens=0, logits=None, dw=None, ids=None, out=None) == OK


def layout_desc(**kw):
    d = _lib.RouteLayoutDesc()
    base = dict(ids=P, ids_64=1, top_k=2, tokens=100, experts=8, alignment=128, rows=200 + 8 * 127, pair_row=P, row_token=P, rows_per_expert=P, offsets=P,
                expert_list=P)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


def test_layout_refuses_bad_descriptors():
    lib = _lib.load()
    assert lib.ag_route_layout(None) == BAD
    for bad in (dict(tokens=-1), dict(top_k=0), dict(experts=0), dict(experts=1025), dict(max_rows=-1), dict(rows=-1), dict(tokens=1 << 31), dict(ids=P + 4),
                dict(pair_row=P + 4), dict(row_token=P + 4), dict(offsets=P + 2), dict(ids=None), dict(pair_row=None), dict(row_token=None), dict(alignment=0),
                dict(rows_per_expert=None), dict(offsets=None), dict(expert_list=None), dict(rows=200 + 8 * 127 - 1),
                dict(max_rows=16, rows=8 * 16), dict(max_rows=16, rows=8 * 16 - 1, masked_m=P), dict(max_rows=16, rows=8 * 17, masked_m=P),
                dict(tokens=5000, rows=10000 + 8 * 127)):      # the last one: several blocks and no workspace
        assert lib.ag_route_layout(layout_desc(**bad)) == BAD, bad
    for tokens in (1 << 62, (1 << 63) - 1):      # tokens * top_k does not fit in 64 bits
        assert lib.ag_route_layout(layout_desc(tokens=tokens)) == BAD
    assert lib.ag_route_layout_workspace_bytes(2048, 256) == 0 and lib.ag_route_layout_workspace_bytes(2049, 254) == 3 * 256 * 4
    assert lib.ag_route_layout_workspace_bytes(0, 8) == 0 and lib.ag_route_layout_workspace_bytes(-5, 8) == 0


def test_combine_gradient_refuses_bad_arguments():
    lib = _lib.load()

    def call(dy=P, rows=P, num_rows=16, pos=P, w=P, tokens=4, k=2, cols=64, drows=P, dw=P, seen=P):
        return lib.ag_combine_topk_backward(dy, rows, 0, num_rows, pos, w, tokens, k, cols, drows, dw, seen, None, None)

    for bad in (dict(tokens=-1), dict(k=0), dict(num_rows=-1), dict(cols=0), dict(cols=60), dict(cols=1 << 31), dict(dy=P + 8), dict(rows=P + 8), dict(drows=P + 8),
                dict(pos=P + 4), dict(w=P + 2), dict(dw=P + 2), dict(seen=P + 2), dict(seen=None), dict(dy=None), dict(w=None), dict(rows=None)):
        assert call(**bad) == BAD, bad
    assert call(drows=None, dw=None, seen=None) == OK and call(tokens=0, drows=None) == OK


def linear_desc(**kw):
    d = _lib.LinearDesc()
    base = dict(m=16, n=32, k=64, x=P, weight=P, y=P, ldx=64, ldw=64, ldy=32)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


def test_dense_product_refuses_bad_descriptors():
    lib = _lib.load()
    assert lib.ag_linear(None) == BAD and lib.ag_linear_backward(None) == BAD
    assert lib.ag_linear_desc_size() == ctypes.sizeof(_lib.LinearDesc)
    common = (dict(dtype=2), dict(out_dtype=1), dict(bias_dtype=1), dict(activation=4), dict(activation=-1), dict(m=-1), dict(n=0), dict(k=0), dict(k=60, ldx=60, ldw=60),
              dict(ldx=56), dict(ldx=68), dict(ldw=56), dict(ldw=68), dict(x=P + 8), dict(weight=P + 2), dict(m=1 << 31), dict(k=1 << 31, ldx=1 << 31, ldw=1 << 31))
    for bad in common + (dict(x=None), dict(weight=None), dict(y=None), dict(ldy=31), dict(residual=P, ldr=31), dict(pre=P, ldp=31), dict(y=P + 1),
                         dict(out_dtype=2, y=P + 2), dict(residual=P + 1, ldr=32), dict(bias=P + 1), dict(bias=P + 2, bias_dtype=2), dict(pre=P + 1, ldp=32)):
        assert lib.ag_linear(linear_desc(**bad)) == BAD, bad
    assert lib.ag_linear(linear_desc(m=0, x=None)) == OK
    back = dict(dy=P, lddy=32, dx=P, dweight=P, dbias=P)
    for bad in common + (dict(x=None), dict(weight=None), dict(dy=None), dict(lddy=31), dict(activation=2), dict(activation=2, pre=P, ldp=31), dict(dx=P + 1),
                         dict(dbias=P + 1), dict(dy=P + 1)):
        assert lib.ag_linear_backward(linear_desc(**{**back, **bad})) == BAD, bad
    assert lib.ag_linear_backward(linear_desc(dy=P, lddy=32)) == OK      # nothing is wanted
    assert lib.ag_linear_workspace_bytes(linear_desc(m=0), 0) == 0 and lib.ag_linear_workspace_bytes(linear_desc(k=60), 1) == 0


def test_python_entry_points_refuse_cpu_tensors_and_unknown_names():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    for call in (lambda: dense_ops.linear(x, w), lambda: dense_ops.linear(x, w, activation="swish"), lambda: dense_ops.linear(x, w, out_dtype=torch.float16),
                 lambda: dense_ops.linear_backward(x, x, w), lambda: moe_ops.route_topk(torch.zeros(4, 8), 2), lambda: moe_ops.route_topk(torch.zeros(4, 8), 2, scoring="tanh"),
                 lambda: moe_ops.route_topk(torch.zeros(4, 8), 2, num_groups=2, group_score="sum"), lambda: moe_ops.route_layout(torch.zeros(4, 2, dtype=torch.int64), 8),
                 lambda: moe_ops.route_layout_masked(torch.zeros(4, 2, dtype=torch.int64), 8, 4),
                 lambda: moe_ops.combine_topk_backward(x, x, None, torch.zeros(4, 1))):
        with pytest.raises(RuntimeError):
            call()


def test_cpu_row_moves_and_combine_skip_what_has_no_row():
    src = torch.arange(12.0).view(4, 3)
    out = moe_ops.move_rows(src, 5, src_rows=torch.tensor([3, -1, 0, 2, -1]))
    assert out.tolist() == [src[3].tolist(), [0, 0, 0], src[0].tolist(), src[2].tolist(), [0, 0, 0]]
    out = moe_ops.move_rows(src, 3, dst_rows=torch.tensor([2, -1, 0, -1]), zero=True)
    assert out.tolist() == [src[2].tolist(), [0, 0, 0], src[0].tolist()]
    y = moe_ops.combine_topk(src, torch.tensor([0, -1, 3, 1]), torch.tensor([[0.5, 9.0], [1.0, 2.0]]), 2, 2)
    assert torch.equal(y, torch.stack([0.5 * src[0], src[3] + 2 * src[1]]))
    assert moe_ops.combine_topk(src, torch.zeros(0, dtype=torch.int64), torch.zeros(0, 2), 0, 2).shape == (0, 3)
