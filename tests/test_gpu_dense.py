"""The dense product with bias, activation and residual, and its gradients, against plain restatements in 64 bits.

Tolerances. `ACC`: the tensor core truncates when it adds 16 products to its fp32 accumulator, at most one step (2^-23) of the
magnitudes summed per addition, over runs of 512 terms (32 additions; 8 more cover the additions inside one instruction); the
runs are joined by rounded additions (2^-24 each, one per run). All relative to the sum of the terms' magnitudes. A rounding to
type t is off by half a step, finfo(t).eps / 2."""
import math

import pytest
import torch

import asymgemm_b200 as ag
from asymgemm_b200 import dense_ops, moe_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def acc(k):
    return 40 * 2 ** -23 + math.ceil(k / 512) * 2 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest step of the type: what a rounding below its normal range can be off by."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def randn(*shape, seed=0, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def act64(z, name):
    if name == "relu":
        return torch.relu(z)
    if name == "gelu":
        return torch.nn.functional.gelu(z)
    return torch.nn.functional.silu(z) if name == "silu" else z


def slope64(z, name):
    z = z.detach().requires_grad_(True)
    return torch.autograd.grad(act64(z, name).sum(), z)[0] if name != "none" else torch.ones_like(z)


def check_forward(x, w, bias=None, activation="none", residual=None, out_dtype=None):
    y, pre = dense_ops.linear(x, w, bias=bias, activation=activation, residual=residual, out_dtype=out_dtype, return_pre=True)
    k = x.shape[-1]
    xd, wd = x.double().reshape(-1, k), w.double()
    z = xd @ wd.t()
    size = xd.abs() @ wd.abs().t()
    off = size * acc(k)
    if bias is not None:
        z = z + bias.double()
        off = off + z.abs() * 2 ** -24
    if pre is not None:
        assert pre.dtype == x.dtype and pre.shape == y.shape
        assert bool(((pre.double().reshape(z.shape) - z).abs() <= off + z.abs() * half(x.dtype) + tiny(x.dtype)).all())
    a = act64(z, activation)
    # |act'| <= 1.13; erfc, exp and the products around them: below 16 roundings of a value |z| or less
    off = 1.13 * off + (a.abs() + z.abs() * 2 ** -2) * 16 * 2 ** -24 * (activation in ("gelu", "silu"))
    if residual is not None:
        a = a + residual.double().reshape(a.shape)
        off = off + a.abs() * 2 ** -24
    got = y.double().reshape(a.shape)
    assert y.dtype == (out_dtype or x.dtype) and y.shape == x.shape[:-1] + (w.shape[0],)
    assert bool(((got - a).abs() <= off + a.abs() * half(y.dtype) + tiny(y.dtype)).all()), float(((got - a).abs() - off - a.abs() * half(y.dtype)).max())
    ag.check_status()
    return y, pre


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 8), (1, 256, 7168), (2, 7, 72), (15, 100, 64), (16, 129, 512), (17, 257, 520), (33, 64, 1000), (64, 512, 2048),
                                   (65, 130, 136), (128, 128, 128), (130, 300, 584), (300, 60, 264), (257, 1030, 72), (1000, 16, 2048)])
def test_product_over_sizes_and_types(m, n, k, dtype):
    x, w = randn(m, k, seed=m, dtype=dtype), randn(n, k, seed=n, dtype=dtype, scale=k ** -0.5)
    check_forward(x, w)
    check_forward(x, w, out_dtype=torch.float32)
    check_forward(x, w, bias=randn(n, seed=1, dtype=dtype), activation="gelu", residual=randn(m, n, seed=2, dtype=dtype))
    check_forward(x, w, bias=randn(n, seed=1, dtype=torch.float32), activation="silu", residual=randn(m, n, seed=2, dtype=torch.float32), out_dtype=torch.float32)


@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "silu"])
def test_epilogues(activation):
    for m, n, k in ((5, 200, 256), (200, 136, 96)):
        x, w = randn(m, k, seed=3), randn(n, k, seed=4, scale=3 * k ** -0.5)
        for bias in (None, randn(n, seed=5), randn(n, seed=5, dtype=torch.float32)):
            for residual in (None, randn(m, n, seed=6)):
                check_forward(x, w, bias, activation, residual)


def test_products_large_enough_for_every_tile():
    for m, n, k in ((2048, 2304, 512), (700, 8200, 320), (4100, 264, 1024), (96, 7168, 2048), (48, 4096, 7168), (20, 1000, 8192)):
        x, w = randn(m, k, seed=m), randn(n, k, seed=n, scale=k ** -0.5)
        check_forward(x, w, bias=randn(n, seed=7), activation="silu")
        check_forward(x, w, out_dtype=torch.float32)


def test_long_sums_of_one_sign_do_not_drift():
    """Accumulated in the tensor core alone these are 2.8e-5 off at k = 7168."""
    for m, n in ((4, 256), (300, 512)):
        x, w = randn(m, 7168, seed=8).abs(), randn(n, 7168, seed=9).abs()
        y = dense_ops.linear(x, w, out_dtype=torch.float32).double()
        want = x.double() @ w.double().t()
        assert bool(((y - want).abs() <= want * acc(7168)).all())


def test_strides_views_leading_dimensions_and_empty_batches():
    wide = randn(70, 600, seed=10)
    x = wide[::2, 8:8 + 136]
    with pytest.raises(RuntimeError, match="16-byte"):       # rows 600 bytes apart do not all start on 16-byte boundaries
        dense_ops.linear(x, randn(90, 300, seed=11)[:, 16:16 + 136])
    w = randn(90, 304, seed=11)[:, 16:16 + 136]
    res = randn(35, 200, seed=12)[:, 3:93]
    check_forward(x, w, residual=res, activation="relu")
    check_forward(randn(3, 5, 64, seed=13), randn(33, 64, seed=14), residual=randn(3, 5, 33, seed=15), activation="gelu")
    check_forward(randn(64, seed=13), randn(33, 64, seed=14))
    y = dense_ops.linear(torch.empty((0, 64), dtype=torch.bfloat16, device=DEV), randn(33, 64, seed=14))
    assert y.shape == (0, 33)
    # the residual may be what the result is added to by name only: the output is a new tensor
    r = randn(35, 90, seed=16)
    kept = r.clone()
    dense_ops.linear(x.contiguous(), w.contiguous(), residual=r)
    assert torch.equal(r, kept)


def test_values_without_end_stay_in_their_rows_and_columns():
    x, w = randn(40, 256, seed=17), randn(70, 256, seed=18)
    x[3, 5], x[9, 0] = math.inf, math.nan
    w[11, 7] = math.nan
    y = dense_ops.linear(x, w, activation="relu")
    clean_x, clean_w = x.clone(), w.clone()
    clean_x[3, 5] = clean_x[9, 0] = clean_w[11, 7] = 0
    want = dense_ops.linear(clean_x, clean_w, activation="relu")
    keep_r = torch.tensor([i not in (3, 9) for i in range(40)], device=DEV)
    keep_c = torch.tensor([i != 11 for i in range(70)], device=DEV)
    assert torch.equal(y[keep_r][:, keep_c], want[keep_r][:, keep_c])
    assert bool(torch.isnan(y[9]).all()) and bool(torch.isnan(y[:, 11]).all())


# ------------------------------------------------------------------------------------------------------ gradients
def check_backward(x, w, dy, activation="none", bias_dtype=None, pre=None):
    dx, dw, db = dense_ops.linear_backward(dy, x, w, activation=activation, pre=pre, bias_dtype=bias_dtype)
    k, n = x.shape[-1], w.shape[0]
    xd, wd, g = x.double().reshape(-1, k), w.double(), dy.double().reshape(-1, n)
    dz = g * slope64(pre.double().reshape(-1, n), activation) if activation != "none" else g
    # the slope: erfc, exp and a few products; then the rounding of dz to the operands' type
    slope_off = g.abs() * 24 * 2 ** -24 * (activation in ("gelu", "silu"))
    dz_off = slope_off + dz.abs() * half(x.dtype) * (activation != "none" or dy.dtype != x.dtype) + tiny(x.dtype)
    m = xd.shape[0]
    for got, want, size, err, terms in ((dx, dz @ wd, dz.abs() @ wd.abs(), dz_off @ wd.abs(), n), (dw, dz.t() @ xd, dz.abs().t() @ xd.abs(), dz_off.t() @ xd.abs(), m)):
        got = got.double().reshape(want.shape)
        bound = size * acc(terms) + err * (1 + 2 ** -7) + want.abs() * half(x.dtype) + tiny(x.dtype)
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())
    want = dz.sum(0)
    # a thread adds at most a block's rows / 8, then 8 and the blocks / 8 and 8 are joined: fewer than m / 8 + 100 additions
    bound = dz.abs().sum(0) * (m / 8 + 100) * 2 ** -24 + slope_off.sum(0) + want.abs() * half(db.dtype) + tiny(db.dtype)
    assert db.dtype == (bias_dtype or x.dtype) and bool(((db.double() - want).abs() <= bound).all())
    assert dx.shape == x.shape and dw.shape == w.shape and db.shape == (n,)
    ag.check_status()
    return dx, dw, db


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 8), (1, 256, 512), (2, 7, 72), (16, 100, 64), (17, 257, 520), (64, 512, 264), (65, 130, 136), (130, 300, 584),
                                   (300, 60, 264), (1000, 16, 1000), (2500, 264, 128)])
def test_gradients_over_sizes_and_types(m, n, k, dtype):
    x, w = randn(m, k, seed=m, dtype=dtype), randn(n, k, seed=n, dtype=dtype, scale=2 * k ** -0.5)
    check_backward(x, w, randn(m, n, seed=20, dtype=dtype))
    check_backward(x, w, randn(m, n, seed=21, dtype=torch.float32), bias_dtype=torch.float32)
    for activation in ("relu", "gelu", "silu"):
        pre = randn(m, n, seed=22, dtype=dtype, scale=2.0)
        check_backward(x, w, randn(m, n, seed=23, dtype=dtype), activation, pre=pre)
        check_backward(x, w, randn(m, n, seed=23, dtype=torch.float32), activation, torch.float32, pre=pre)


def test_gradients_large_enough_for_every_tile():
    for m, n, k in ((2048, 2304, 1024), (16384, 256, 2048), (4100, 1030, 520), (3000, 8, 8)):
        x, w = randn(m, k, seed=m), randn(n, k, seed=n, scale=k ** -0.5)
        check_backward(x, w, randn(m, n, seed=24), "silu", pre=randn(m, n, seed=25))
        check_backward(x, w, randn(m, n, seed=24))


def test_gradients_of_views_and_of_parts():
    m, n, k = 70, 96, 136
    x, w = randn(2 * m, 600, seed=26)[::2, 8:8 + k], randn(n, 304, seed=27)[:, 16:16 + k]
    for dy in (randn(m, 300, seed=28)[:, 3:3 + n], randn(m, 200, seed=28)[:, 8:8 + n], randn(3 * m, n, seed=28)[::3]):
        all_three = check_backward(x, w, dy)
        for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (False, False, False)):
            some = dense_ops.linear_backward(dy, x, w, need_x=need[0], need_weight=need[1], need_bias=need[2])
            for got, want, wanted in zip(some, all_three, need):
                assert torch.equal(got, want) if wanted else got is None
    dx, dw, db = dense_ops.linear_backward(dy[:0], x[:0], w)
    assert dx.shape == (0, k) and float(dw.abs().max()) == 0 and float(db.abs().max()) == 0


@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "silu"])
def test_autograd_gives_the_same_gradients(activation):
    x, w, b, r = randn(4, 9, 72, seed=30), randn(50, 72, seed=31, scale=0.3), randn(50, seed=32, dtype=torch.float32), randn(4, 9, 50, seed=33)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    y = dense_ops.linear(leaves[0], leaves[1], bias=leaves[2], activation=activation, residual=leaves[3])
    again, pre = dense_ops.linear(x, w, bias=b, activation=activation, residual=r, return_pre=True)
    assert torch.equal(y, again)
    dy = randn(4, 9, 50, seed=34)
    got = torch.autograd.grad(y, leaves, dy)
    want = dense_ops.linear_backward(dy, x, w, activation=activation, pre=pre, bias_dtype=torch.float32)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(got[3], dy)
    # a gradient that is one number everywhere, and one laid out the other way round
    y = dense_ops.linear(leaves[0].reshape(36, 72), leaves[1], activation=activation)
    y.sum().backward()
    plain = torch.autograd.grad(dense_ops.linear(leaves[0].reshape(36, 72), leaves[1], activation=activation), leaves[1], torch.ones(36, 50, device=DEV, dtype=torch.bfloat16))
    assert torch.equal(leaves[1].grad, plain[0])
    y = dense_ops.linear(leaves[0], leaves[1], activation=activation)
    wide = torch.autograd.grad(y, leaves[1], torch.ones((1, 1, 50), device=DEV, dtype=torch.bfloat16).expand(4, 9, 50))
    assert torch.equal(wide[0], plain[0])
    y = dense_ops.linear(leaves[0].reshape(36, 72), leaves[1], activation=activation)
    turned = torch.autograd.grad(y, leaves[1], randn(50, 36, seed=35).t(), retain_graph=True)[0]
    straight = torch.autograd.grad(y, leaves[1], randn(50, 36, seed=35).t().contiguous())[0]
    assert torch.equal(turned, straight)


@pytest.mark.parametrize("activation", ["gelu", "silu", "relu"])
def test_gradient_against_differences(activation):
    """The formulas of the slopes, by central differences in 64 bits at the operands the kernel has."""
    z = torch.cat([torch.linspace(-6, 6, 97) + 0.01, torch.tensor([-20.0, 20.0, -0.3, 0.3])]).to(torch.float16)
    n = z.numel()
    pre = z.view(1, n).to(DEV)
    x, w = torch.ones((1, 8), dtype=torch.float16, device=DEV), torch.zeros((n, 8), dtype=torch.float16, device=DEV)
    dy = torch.ones((1, n), dtype=torch.float32, device=DEV)
    db = dense_ops.linear_backward(dy, x, w, activation=activation, pre=pre, need_x=False, need_weight=False, bias_dtype=torch.float32)[2]
    zd, step = z.double(), 1e-6
    num = (act64(zd + step, activation) - act64(zd - step, activation)) / (2 * step)
    # third derivatives below 3, so step^2 / 2; 64-bit rounding of values up to 20 over the step; fp32 slope
    assert torch.allclose(db.cpu().double(), num, rtol=0, atol=20 * 2 ** -52 / step + 24 * 2 ** -24)


# ------------------------------------------------------------------------------------------------------ use
def test_refusals():
    x, w = randn(16, 64), randn(32, 64)
    for args, kw in (((x.cpu(), w), {}), ((x, w.cpu()), {}), ((x.float(), w.float()), {}), ((x, w.half()), {}), ((x, randn(32, 72)), {}), ((x, randn(64)), {}),
                     ((randn(16, 60), randn(32, 60)), {}), ((x.t(), randn(32, 16)), {}), ((randn(16, 200)[:, 4:68], w), {}), ((randn(16, 66)[:, :64], w), {}),
                     ((x, w), dict(bias=randn(31))), ((x, w), dict(bias=randn(32, dtype=torch.float16))), ((x, w), dict(bias=randn(32).cpu())),
                     ((x, w), dict(residual=randn(16, 31))), ((x, w), dict(residual=randn(16, 32, dtype=torch.float32))),
                     ((x, w), dict(residual=randn(16, 32), out_dtype=torch.float32)), ((x, w), dict(activation="tanh")), ((x, w), dict(out_dtype=torch.float16)),
                     ((randn(2, 8, 64), w), dict(residual=randn(16, 32)))):
        with pytest.raises(RuntimeError):
            dense_ops.linear(*args, **kw)
    dy = randn(16, 32)
    for args, kw in (((dy.half(), x, w), {}), ((dy[:, :31], x, w), {}), ((dy[:15], x, w), {}), ((dy, x, w), dict(activation="gelu")),
                     ((dy, x, w), dict(activation="gelu", pre=dy[:, :31])), ((dy, x, w), dict(activation="gelu", pre=dy.float())),
                     ((dy, x, w), dict(bias_dtype=torch.float16)), ((dy.cpu(), x, w), {})):
        with pytest.raises(RuntimeError):
            dense_ops.linear_backward(*args, **kw)
    pinned = torch.empty((32, 64), dtype=torch.bfloat16).pin_memory()
    with pytest.raises(RuntimeError):
        dense_ops.linear(x, pinned)


def test_the_result_may_take_the_residuals_place_through_the_c_abi():
    from asymgemm_b200 import _lib
    lib = _lib.load()
    for m, n, k in ((30, 200, 512), (1000, 1536, 256), (40, 90, 136)):
        x, w, r = randn(m, k, seed=36), randn(n, k, seed=37, scale=k ** -0.5), randn(m, n, seed=38)
        want = dense_ops.linear(x, w, residual=r, activation="silu")
        d = _lib.LinearDesc(m=m, n=n, k=k, activation=3, x=x.data_ptr(), weight=w.data_ptr(), residual=r.data_ptr(), y=r.data_ptr(), ldx=k, ldw=k, ldr=n, ldy=n,
                            stream=torch.cuda.current_stream().cuda_stream)
        space = torch.empty(max(1, int(lib.ag_linear_workspace_bytes(d, 0))), dtype=torch.uint8, device=DEV)
        d.workspace, d.workspace_bytes = space.data_ptr(), space.numel()
        _lib.check(lib.ag_linear(d))
        assert torch.equal(r, want)


def test_two_streams_and_two_captured_graphs_at_once():
    """Products that run side by side share nothing: two graphs with workspaces, replayed on two streams."""
    cases = []
    for i in range(2):
        x, w = randn(900, 520, seed=40 + i), randn(264, 520, seed=50 + i, scale=0.05)
        dy, pre = randn(900, 264, seed=60 + i), randn(900, 264, seed=70 + i)
        cases.append((x, w, dy, pre))

    def step(c):
        x, w, dy, pre = c
        return (dense_ops.linear(x, w, activation="gelu"),) + dense_ops.linear_backward(dy, x, w, activation="gelu", pre=pre)

    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    eager = []
    for c, s in zip(cases, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            eager.append(step(c))
    torch.cuda.synchronize()
    for got, ref in zip(eager, want):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_router_in_training_together():
    """Router weights trained over frozen experts: logits -> route -> layout -> experts (each scales its rows) -> combine with a
    shared expert as residual, and the gradients of the router's weights and of the shared expert against autograd in 64 bits."""
    tokens, experts, k, hidden = 200, 16, 4, 128
    x = randn(tokens, hidden, seed=80)
    gate = randn(experts, hidden, seed=81, scale=hidden ** -0.5).requires_grad_(True)
    up = randn(96, hidden, seed=82, scale=hidden ** -0.5).requires_grad_(True)
    down = randn(hidden, 96, seed=83, scale=96 ** -0.5).requires_grad_(True)
    factor = torch.linspace(0.5, 2.0, experts, device=DEV).to(torch.bfloat16)
    logits = dense_ops.linear(x, gate, out_dtype=torch.float32)
    ids, weights = moe_ops.route_topk(logits, k, scoring="sigmoid", scale=1.5)
    lay = moe_ops.route_layout(ids, experts)
    rows = moe_ops.move_rows(x, lay.row_token.numel(), src_rows=lay.row_token)
    owner = torch.zeros(rows.shape[0], dtype=torch.int64, device=DEV)
    owner[lay.pair_row] = ids.reshape(-1)
    rows = rows * factor[owner].unsqueeze(1)
    routed = moe_ops.combine_topk(rows, lay.pair_row, weights, tokens, k)
    y = dense_ops.linear(dense_ops.linear(x, up, activation="silu"), down, residual=routed)
    dy = randn(tokens, hidden, seed=84)
    got = torch.autograd.grad(y, (gate, up, down), dy)

    leaves = [t.detach().double().requires_grad_(True) for t in (gate, up, down)]
    xd = x.double()
    s = torch.sigmoid(xd @ leaves[0].t()).gather(1, ids)
    w = 1.5 * s / s.sum(1, keepdim=True)
    routed = torch.einsum("tk,th->th", w * factor.double()[ids], xd)
    h = torch.nn.functional.silu(xd @ leaves[1].t())
    want_y = h @ leaves[2].t() + routed
    want = torch.autograd.grad(want_y, leaves, dy.double())
    for a, b in zip((y,) + got, (want_y,) + want):
        # a handful of independent bf16 roundings (2^-9 rms each) on the way: rows, weights' products, h, dz, result
        assert float(((a.double() - b).norm() / b.norm()).detach()) <= 8 * 2 ** -9
    ag.check_status()
