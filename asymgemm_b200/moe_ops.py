"""Python wrappers of the MoE helper kernels (csrc/moe_glue.cu, csrc/route.cu) declared in include/asymgemm_b200.h.

CUDA tensors go through the C ABI (and fail loudly if the library is missing). The row-movement helpers also accept
CPU tensors, where they are plain torch indexing: that branch exists only so that the expert-parallel routing logic can
be exercised by gloo ranks without a GPU; the quantisers, the router and the GEMMs have no CPU branch.

`route_topk` and `combine_topk` are differentiable: with gradients enabled, calls whose logits, rows or weights require
one are recorded for autograd. Their gradients are also functions of their own (`route_topk_backward`,
`combine_topk_backward`), which is the form to capture into a CUDA graph. Forward-mode derivatives exist for `combine_topk` (in plain
torch); the router refuses them.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib, api


def _stream(t: torch.Tensor):
    return torch.cuda.current_stream(t.device).cuda_stream


def quant_rows_fp8(x: torch.Tensor, pow2_scales: bool = False, rows_used: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [rows, cols] -> (e4m3 [rows, cols], fp32 scales [rows, ceil(cols/128)]), one kernel.
    `pow2_scales` rounds the scales up to powers of two (the quantisers' use_ue8m0=True). `rows_used`: device int32 tensor;
    rows from that count on are neither read nor written."""
    if not (x.is_cuda and x.dtype == torch.bfloat16 and x.dim() == 2 and x.is_contiguous()):
        raise RuntimeError("quant_rows_fp8 wants a contiguous 2-D bf16 CUDA tensor")
    rows, cols = x.shape
    q = torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device=x.device)
    sf = torch.empty((rows, (cols + 127) // 128), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ag_quant_rows_fp8_upto(x.data_ptr(), q.data_ptr(), sf.data_ptr(), rows, cols, int(pow2_scales),
                                                      rows_used.data_ptr() if rows_used is not None else None, _stream(x)))
    return q, sf


def silu_mul_quant_fp8(gate_up: torch.Tensor, inter: int, pow2_scales: bool = False,
                       rows_used: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [rows, 2*inter] -> bf16(silu(gate) * up) quantised to (e4m3 [rows, inter], fp32 [rows, ceil(inter/128)]).
    `rows_used`: device int32 tensor; rows from that count on are neither read nor written."""
    if not (gate_up.is_cuda and gate_up.dtype == torch.bfloat16 and gate_up.dim() == 2 and gate_up.is_contiguous()
            and gate_up.shape[1] == 2 * inter):
        raise RuntimeError("silu_mul_quant_fp8 wants a contiguous bf16 CUDA tensor [rows, 2*inter]")
    rows = gate_up.shape[0]
    q = torch.empty((rows, inter), dtype=torch.float8_e4m3fn, device=gate_up.device)
    sf = torch.empty((rows, (inter + 127) // 128), dtype=torch.float32, device=gate_up.device)
    with torch.cuda.device(gate_up.device):
        _lib.check(_lib.load().ag_silu_mul_quant_fp8_upto(gate_up.data_ptr(), q.data_ptr(), sf.data_ptr(), rows, inter, int(pow2_scales),
                                                          rows_used.data_ptr() if rows_used is not None else None, _stream(gate_up)))
    return q, sf


def quant_rows_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [rows, cols] -> (int8 [rows, cols], fp32 [rows, ceil(cols/128)] holding the row's scale in every K-block slot)."""
    if not (x.is_cuda and x.dtype == torch.bfloat16 and x.dim() == 2 and x.is_contiguous()):
        raise RuntimeError("quant_rows_int8 wants a contiguous 2-D bf16 CUDA tensor")
    rows, cols = x.shape
    q = torch.empty((rows, cols), dtype=torch.int8, device=x.device)
    sf = torch.empty((rows, (cols + 127) // 128), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ag_quant_rows_int8(x.data_ptr(), q.data_ptr(), sf.data_ptr(), rows, cols, _stream(x)))
    return q, sf


def silu_mul_quant_int8(gate_up: torch.Tensor, inter: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 [rows, 2*inter] -> bf16(silu(gate) * up) quantised per row to (int8 [rows, inter], fp32 [rows, ceil(inter/128)])."""
    if not (gate_up.is_cuda and gate_up.dtype == torch.float32 and gate_up.dim() == 2 and gate_up.is_contiguous()
            and gate_up.shape[1] == 2 * inter):
        raise RuntimeError("silu_mul_quant_int8 wants a contiguous fp32 CUDA tensor [rows, 2*inter]")
    rows = gate_up.shape[0]
    q = torch.empty((rows, inter), dtype=torch.int8, device=gate_up.device)
    sf = torch.empty((rows, (inter + 127) // 128), dtype=torch.float32, device=gate_up.device)
    with torch.cuda.device(gate_up.device):
        _lib.check(_lib.load().ag_silu_mul_quant_int8(gate_up.data_ptr(), q.data_ptr(), sf.data_ptr(), rows, inter, _stream(gate_up)))
    return q, sf


def _row_bytes(t: torch.Tensor) -> int:
    n = t.element_size()
    for s in t.shape[1:]:
        n *= int(s)
    return n


def _never_empty(rows: torch.Tensor) -> torch.Tensor:
    """`rows`, or one row of zeros where there are none: a table of nothing but -1 (an empty batch in the masked layout) reads none."""
    return rows if rows.shape[0] else torch.cat([rows, rows.new_zeros((1,) + tuple(rows.shape[1:]))])


def move_rows(src: torch.Tensor, out_rows: int, src_rows: Optional[torch.Tensor] = None, dst_rows: Optional[torch.Tensor] = None,
              count: Optional[int] = None, zero: bool = False) -> torch.Tensor:
    """out[dst_rows[i] or i] = src[src_rows[i] or i] for i < count. `out` has `out_rows` rows of src's row shape and dtype.
    A negative src_rows[i] writes a row of zeros, a negative dst_rows[i] writes nothing."""
    count = int(count if count is not None else (src_rows.numel() if src_rows is not None else
                                                 (dst_rows.numel() if dst_rows is not None else src.shape[0])))

    def room(rows):
        return (torch.zeros if zero else torch.empty)((rows,) + tuple(src.shape[1:]), dtype=src.dtype, device=src.device)

    if count == 0:
        return room(out_rows)
    if src_rows is not None:
        src = _never_empty(src)
    rb = _row_bytes(src)
    if src.is_cuda and rb % 16 == 0 and src.is_contiguous():
        out = room(out_rows)
        with torch.cuda.device(src.device):
            _lib.check(_lib.load().ag_move_rows(src.data_ptr(), out.data_ptr(),
                                                src_rows.data_ptr() if src_rows is not None else None,
                                                dst_rows.data_ptr() if dst_rows is not None else None, count, rb, _stream(src)))
        return out
    # plain torch, without waiting for the device: rows without a destination go to one row more, behind the result
    s = src.view(torch.uint8) if src.dtype == torch.float8_e4m3fn else src
    if src_rows is not None:
        src_rows = src_rows[:count]
        picked = s.index_select(0, src_rows.clamp(min=0))
        picked.masked_fill_((src_rows < 0).view((-1,) + (1,) * (s.dim() - 1)), 0)
    else:
        picked = s[:count]
    out = room(out_rows + (dst_rows is not None))
    o = out.view(torch.uint8) if out.dtype == torch.float8_e4m3fn else out
    if dst_rows is None:
        o[:count] = picked
        return out
    dst_rows = dst_rows[:count]
    o.index_copy_(0, torch.where(dst_rows < 0, out_rows, dst_rows), picked)
    return out[:out_rows]


def move_rows_into(out: torch.Tensor, src: torch.Tensor, dst_rows: torch.Tensor) -> None:
    """out[dst_rows[i]] = src[i] for every row of src, in place (rows of out that are not named keep their contents)."""
    count = int(dst_rows.numel())
    if count == 0:
        return
    rb = _row_bytes(src)
    if src.is_cuda and rb % 16 == 0 and src.is_contiguous() and out.is_contiguous():
        with torch.cuda.device(src.device):
            _lib.check(_lib.load().ag_move_rows(src.data_ptr(), out.data_ptr(), None, dst_rows.data_ptr(), count, rb, _stream(src)))
        return
    out.index_copy_(0, dst_rows, src)


def _has_combine_kernel(rows: torch.Tensor) -> bool:
    if not rows.is_cuda:
        return False
    dtype, cols = rows.dtype, rows.shape[1]
    return (cols % 8 == 0 if dtype is torch.bfloat16 else dtype is torch.float32 and cols % 4 == 0) and rows.is_contiguous()


def _check_combine_tables(rows, pos, weights, pairs: int) -> None:
    """What the kernels read by address: wrong types or too few entries would be read past their end."""
    gpu = rows.get_device()
    if pos is None:
        if rows.shape[0] < pairs:
            raise RuntimeError(f"without pos, rows must hold a row for each of the {pairs} slots")
    elif pos.dtype is not torch.int64 or pos.get_device() != gpu or not pos.is_contiguous() or pos.numel() < pairs:
        raise RuntimeError(f"pos must be a contiguous int64 tensor of {pairs} entries at least, on the device of rows")
    if weights.get_device() != gpu or weights.numel() < pairs:
        raise RuntimeError(f"weights must hold {pairs} entries on the device of rows")


def combine_topk(rows: torch.Tensor, pos: torch.Tensor, weights: torch.Tensor, tokens: int, top_k: int) -> torch.Tensor:
    """y[t] = sum_j weights[t, j] * rows[pos[t*top_k + j]] (fp32 accumulation), as rows.dtype (bf16 where a CUDA kernel runs); pos
    None = t*top_k + j. Slots with a negative pos (pairs a layout dropped) add nothing. Differentiable with respect to `rows` and
    `weights`; where the CUDA kernels run (contiguous rows, bf16 or fp32, cols a multiple of 8) the gradient is
    `combine_topk_backward`'s: no two slots may name the same row. Elsewhere it is plain torch's."""
    if api._has_tangent(rows, weights) and _has_combine_kernel(rows):
        return _combine_plain(rows, pos, weights, tokens, top_k).to(torch.bfloat16)      # the kernels have no forward-mode derivative
    if (rows.requires_grad or weights.requires_grad) and torch.is_grad_enabled() and _has_combine_kernel(rows):
        return _CombineTopK.apply(rows, pos, weights, tokens, top_k)
    return combine_topk_forward(rows, pos, weights, tokens, top_k)


def combine_topk_forward(rows: torch.Tensor, pos: torch.Tensor, weights: torch.Tensor, tokens: int, top_k: int) -> torch.Tensor:
    """`combine_topk` without a record for autograd where the CUDA kernels run: the layers' inference path, whose GEMMs have none
    either and whose buffers the next call overwrites."""
    cols = rows.shape[1]
    if not _has_combine_kernel(rows):
        return _combine_plain(rows, pos, weights, tokens, top_k).to(rows.dtype)
    if tokens == 0:
        return torch.empty((0, cols), dtype=torch.bfloat16, device=rows.device)
    if pos is not None:
        rows = _never_empty(rows)
    _check_combine_tables(rows, pos, weights, tokens * top_k)
    if rows.dtype == torch.float32 and pos is None:
        pos = torch.arange(tokens * top_k, device=rows.device)
    y = torch.empty((tokens, cols), dtype=torch.bfloat16, device=rows.device)
    w = weights if weights.dtype is torch.float32 and weights.is_contiguous() else weights.to(torch.float32).contiguous()
    with torch.cuda.device(rows.device):
        combine = _lib.load().ag_combine_topk if rows.dtype == torch.bfloat16 else _lib.load().ag_combine_topk_f32
        _lib.check(combine(rows.data_ptr(), pos.data_ptr() if pos is not None else None, w.data_ptr(), y.data_ptr(), tokens, top_k, cols, _stream(rows)))
    return y


def _combine_plain(rows, pos, weights, tokens: int, top_k: int) -> torch.Tensor:
    """The sum in plain torch, fp32: types and widths without a kernel, and CPU tensors."""
    if pos is None:
        return (rows[: tokens * top_k].reshape(tokens, top_k, rows.shape[1]).float() * weights.reshape(tokens, top_k, 1).float()).sum(dim=1)
    pos = pos.reshape(-1)[: tokens * top_k]      # a table may be longer than the batch
    none = (pos < 0).view(tokens, top_k, 1)      # what has no row adds nothing, whatever its weight and row 0 are
    picked = _never_empty(rows).index_select(0, pos.clamp(min=0)).view(tokens, top_k, rows.shape[1])
    return (picked.float().masked_fill(none, 0) * weights.reshape(tokens, top_k, 1).float().masked_fill(none, 0)).sum(dim=1)


def combine_topk_backward(dy: torch.Tensor, rows: torch.Tensor, pos: Optional[torch.Tensor], weights: torch.Tensor, need_rows: bool = True,
                          need_weights: bool = True) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients of `combine_topk` from dy bf16 [tokens, cols]: (drows like rows, dweights fp32 [tokens, top_k]), None for one
    that is not needed (frozen experts need dweights only, which leaves the rows' half of the memory traffic out).

    dweights[t, j] = <dy[t], rows[pos]> in fp32; drows[pos] = weights[t, j] * dy[t], rounded once, and 0 in rows that no
    slot names. Slots with a pos outside the rows add nothing. With `need_rows` a row may be named by one slot only, as every
    layout here does: a second one sets the status word (`check_status` raises). cols must be a multiple of 8."""
    api._refuse_tangents(dy, rows, weights)
    w = weights if weights.dtype == torch.float32 and weights.is_contiguous() else weights.to(torch.float32).contiguous()
    return _lib.torch_ops().combine_topk_backward(dy, rows, pos, w, bool(need_rows), bool(need_weights), api._status_word(dy.device))


class _CombineTopK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, pos, weights, tokens, top_k):
        ctx.save_for_backward(rows, pos, weights)
        ctx.top_k = top_k
        return combine_topk_forward(rows, pos, weights, tokens, top_k)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rows, pos, weights = ctx.saved_tensors
        if rows.shape[1] % 8:      # fp32 rows of 4 mod 8 columns: the forward pass has a kernel, the gradient has none
            with torch.enable_grad():
                leaves = [rows.detach().requires_grad_(True), weights.detach().requires_grad_(True)]
                y = _combine_plain(leaves[0], pos, leaves[1], dy.shape[0], ctx.top_k)
            grads = torch.autograd.grad(y, [t for t, need in zip(leaves, (ctx.needs_input_grad[0], ctx.needs_input_grad[2])) if need], dy.float())
            return grads[0] if ctx.needs_input_grad[0] else None, None, grads[-1] if ctx.needs_input_grad[2] else None, None, None
        if pos is not None:
            pos = pos[: weights.numel()]      # a table may be longer than the batch
        drows, dweights = combine_topk_backward(dy.contiguous(), rows, pos, weights.reshape(dy.shape[0], ctx.top_k), ctx.needs_input_grad[0],
                                                ctx.needs_input_grad[2])
        if dweights is not None:
            dweights = dweights.view(weights.shape).to(weights.dtype)
        return drows, None, dweights, None, None


# --------------------------------------------------------------------------------------------- routing
MAX_LAYOUT_EXPERTS = 1024      # experts that route_layout builds tables for
_SCORING = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORE = {"top2": False, "max": True}


def _named(table: dict, name: str, what: str):
    if name not in table:
        raise RuntimeError(f"{what} must be one of {', '.join(map(repr, table))}, got {name!r}")
    return table[name]


def route_topk(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, num_groups: int = 1,
               top_groups: int = 1, group_score: str = "top2", renormalize: bool = True, scale: float = 1.0,
               rows_used: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Router: logits [tokens, experts] (bf16, fp16 or fp32; rows may be strided) -> (topk_ids int64, topk_weights fp32), both
    [tokens, top_k], largest first: what `ExpertParallelMoE.forward`, `Int8MoELayer.forward` and `route_layout` take.

    Scores are `softmax` over all experts or `sigmoid`. Experts are chosen by score + `bias` (fp32 [experts], a
    balance term that does not enter the weights), the lowest index among equals; with `num_groups` > 1 only among the
    `top_groups` groups of consecutive experts whose two largest (`group_score="top2"`) or largest ("max") such values
    are best. Weights are the chosen experts' scores, divided by their sum (`renormalize`), times `scale`.

    The order is that of exact arithmetic: fp32 scores too close to tell apart are compared in fp64. A NaN or -inf logit or
    bias switches an expert off for the token, a +inf logit counts as the largest finite number. Slots for which no expert is
    left, and all slots of tokens from `rows_used` on (device int32 tensor of one element: a batch padded at its end), get id
    -1 and weight 0; `route_layout` and `combine_topk` skip them. At most 1024 experts, 32 groups, top_k 32. Ids and weights lie
    side by side in one allocation, which each of them keeps.

    Differentiable with respect to `logits` through the weights (`route_topk_backward`)."""
    api._refuse_tangents(logits, bias)
    args = (int(top_k), _named(_SCORING, scoring, "scoring"), bias, int(num_groups), int(top_groups),
            _named(_GROUP_SCORE, group_score, "group_score"), bool(renormalize), float(scale), rows_used)
    if logits.requires_grad and torch.is_grad_enabled():
        return _RouteTopK.apply(logits, *args)
    return _lib.torch_ops().route_topk(logits, *args)


def route_topk_backward(dweights: torch.Tensor, topk_ids: torch.Tensor, logits: torch.Tensor, scoring: str = "softmax", renormalize: bool = True,
                        scale: float = 1.0) -> torch.Tensor:
    """dlogits [tokens, experts] (type of `logits`) from dweights fp32 [tokens, top_k], the `topk_ids` that `route_topk` chose
    and its arguments. The choice has no gradient; slots with id -1 add nothing."""
    api._refuse_tangents(dweights, logits)
    return _lib.torch_ops().route_topk_backward(dweights, topk_ids, logits, _named(_SCORING, scoring, "scoring"), bool(renormalize), float(scale))


class _RouteTopK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, *args):
        ids, weights = _lib.torch_ops().route_topk(logits, *args)
        ctx.save_for_backward(logits, ids)
        ctx.how = (args[1], args[6], args[7])
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, dweights):
        logits, ids = ctx.saved_tensors
        dlogits = _lib.torch_ops().route_topk_backward(dweights.to(torch.float32).contiguous(), ids, logits, *ctx.how)
        return (dlogits,) + (None,) * 9


class RouteLayout(NamedTuple):
    """Tables of the contiguous layout (`route_layout`). They lie side by side in one allocation (one takes the host less time than
    five): each keeps the memory of all, and `torch.save` writes all, so clone what outlives the step, e.g. `rows_per_expert`."""
    pair_row: torch.Tensor         # int64 [tokens * top_k]: row of every (token, slot) pair, -1 = none (`pos` of combine_topk)
    row_token: torch.Tensor        # int64 [rows]: token of every row, -1 = padding (`src_rows` of move_rows)
    rows_per_expert: torch.Tensor  # int64 [experts]
    offsets: torch.Tensor          # int32 [2 * experts]: (start, end) of every expert's padded segment
    experts: torch.Tensor          # int32 [experts + 1]: 0 .. experts - 1, -1


class MaskedRouteLayout(NamedTuple):
    """Tables of the masked layout (`route_layout_masked`); one allocation, as for `RouteLayout`."""
    pair_row: torch.Tensor         # int64 [tokens * top_k]: row in the flattened [experts * max_rows], -1 = none or dropped
    row_token: torch.Tensor        # int64 [experts * max_rows]: token of every row, -1 = unused
    masked_m: torch.Tensor         # int32 [experts]: rows used


def route_layout(topk_ids: torch.Tensor, num_experts: int, alignment: int = 128) -> RouteLayout:
    """Tables of the contiguous layout of the grouped GEMMs from topk_ids [tokens, top_k] (int64 or int32, CUDA), on the device
    and without a host synchronisation: pairs sorted by expert, in their own order within one, every expert's segment padded to
    `alignment` rows. `row_token` has room for the worst case (all pairs plus one alignment per expert), -1 past the last row.
    Ids of -1 (no expert) get no row; other ids outside [0, num_experts) do neither and set the status word (`check_status`
    raises). At most 1024 experts."""
    return RouteLayout(*_lib.torch_ops().route_layout(topk_ids, int(num_experts), int(alignment), api._status_word(topk_ids.device)))


def route_layout_masked(topk_ids: torch.Tensor, num_experts: int, max_rows: int) -> MaskedRouteLayout:
    """As `route_layout` for the masked layout: expert e has the rows e * max_rows ... of [num_experts, max_rows]. Pairs that find
    their expert's rows taken are dropped (row -1; first come, first served in token order), as a router with a capacity does."""
    return MaskedRouteLayout(*_lib.torch_ops().route_layout_masked(topk_ids, int(num_experts), int(max_rows), api._status_word(topk_ids.device)))
