"""torch.library custom ops over the MI355X MoE kernels (namespace ``moe_mi355x``; those on
block-scaled 4-bit operands and 8-bit kept activations ``moe_mi355x_mx``, those on 8-bit integers
``moe_mi355x_int8``).

Each op is a thin host wrapper around one C-ABI entry point of
``libmoe_mi355x.so``: it allocates outputs and workspaces with torch's caching
allocator, passes raw device pointers and torch's current stream, and maps
status codes to exceptions. Every op has a fake (meta) implementation so it
stays opaque under ``torch.compile``, and an autograd formula, following the
registration pattern of torchtitan/ops/scatter_add.py:10-48.

There is no CPU or eager-torch fallback: the ops raise on non-GPU tensors and
when the library is missing.
"""

from __future__ import annotations

import functools
from contextlib import nullcontext

import torch
from torch import Tensor
from torch.autograd import forward_ad

from ._lib import call, lib, ptr, require_gpu, stream_of

SCORE_FUNCS = {"softmax": 0, "sigmoid": 1}
# Shape limits of the routing kernels taken together: the router takes E <= 512
# and K <= 64, the histogram and reorder K <= 32 (and E <= 1024).
MAX_EXPERTS = 512
MAX_TOP_K = 32
MAX_GEMM_EXPERTS = 1024  # of the grouped GEMMs
DTYPE_CODES = {torch.bfloat16: 0, torch.float32: 1}

# Gradient of x[token_idx] accumulates a token's K rows with a rounding to the
# row dtype after each add, as ATen's index_put(accumulate=True) kernel does for
# row slices on the GPU.
PERMUTE_BWD_ROUND_EACH = True


def _dtype_code(t: Tensor) -> int:
    try:
        return DTYPE_CODES[t.dtype]
    except KeyError:
        raise TypeError(f"MoE row kernels support bfloat16 and float32 rows, got {t.dtype}") from None


def _workspace(n_tokens: int, num_experts: int, device: torch.device) -> Tensor:
    nbytes = lib().moe_reorder_workspace_bytes(n_tokens, num_experts)
    return torch.empty(max(nbytes, 4), dtype=torch.uint8, device=device)


# ---------------------------------------------------------------------------
# router: score function, bias, group limit, top-k, gather, norm, scale
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::router", mutates_args=())
def router(
    logits: Tensor,
    expert_bias: Tensor | None,
    num_experts: int,
    top_k: int,
    score_func: int,
    num_expert_groups: int,
    num_limited_groups: int,
    route_norm: bool,
    route_scale: float,
    force_load_balance: bool,
    with_counts: bool = True,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Returns (top_scores [N,K] f32, selected_experts [N,K] i64, counts [E] i64, scores [N,E] f32).
    with_counts=False skips the histogram (moe.py:269-274) and returns an empty counts
    tensor, for callers that take the counts from the reorder that follows (its own
    histogram, moe.py:312-317, the same counts on one GPU)."""
    require_gpu(logits, expert_bias)
    logits = logits.float().contiguous()
    n = logits.shape[0]
    dev = logits.device
    bias = expert_bias.float().contiguous() if expert_bias is not None else None
    scores = torch.empty_like(logits)
    top_scores = torch.empty(n, top_k, dtype=torch.float32, device=dev)
    idx = torch.empty(n, top_k, dtype=torch.int64, device=dev)
    counts = torch.empty(num_experts if with_counts else 0, dtype=torch.int64, device=dev)
    s = stream_of(logits)
    call(
        "moe_router_fwd", ptr(logits), ptr(bias), n, num_experts, top_k, score_func, num_expert_groups,
            num_limited_groups, int(route_norm), route_scale, int(force_load_balance),
            ptr(scores), ptr(top_scores), ptr(idx), s,
    )
    if with_counts:
        ws = _workspace(n, num_experts, dev)
        call(
            "moe_histogram", ptr(idx), n, top_k, num_experts, ptr(ws), ws.numel(), ptr(counts), None, s
        )
    return top_scores, idx, counts, scores


@router.register_fake
def _(logits, expert_bias, num_experts, top_k, score_func, num_expert_groups, num_limited_groups,
      route_norm, route_scale, force_load_balance, with_counts=True):
    n = logits.shape[0]
    return (
        logits.new_empty(n, top_k, dtype=torch.float32),
        logits.new_empty(n, top_k, dtype=torch.int64),
        logits.new_empty(num_experts if with_counts else 0, dtype=torch.int64),
        logits.new_empty(logits.shape, dtype=torch.float32),
    )


@torch.library.custom_op("moe_mi355x::router_backward", mutates_args=())
def router_backward(
    grad_top_scores: Tensor, scores: Tensor, selected_experts: Tensor, score_func: int,
    route_norm: bool, route_scale: float,
) -> Tensor:
    require_gpu(grad_top_scores, scores, selected_experts)
    g = grad_top_scores.float().contiguous()
    n, e = scores.shape
    k = selected_experts.shape[1]
    out = torch.empty_like(scores)
    call(
        "moe_router_bwd", ptr(g), ptr(scores), ptr(selected_experts), n, e, k, score_func,
                             int(route_norm), route_scale, ptr(out), stream_of(scores)
    )
    return out


@router_backward.register_fake
def _(grad_top_scores, scores, selected_experts, score_func, route_norm, route_scale):
    return torch.empty_like(scores)


def _router_setup(ctx, inputs, output):
    (_logits, _bias, _e, _k, score_func, _g, _gk, route_norm, route_scale, _flb, _wc) = inputs
    _top, idx, counts, scores = output
    ctx.save_for_backward(scores, idx)
    ctx.cfg = (score_func, route_norm, route_scale)
    ctx.mark_non_differentiable(idx, counts, scores)
    ctx.set_materialize_grads(False)  # no zero-filled grads for the index / saved outputs


def _router_bwd(ctx, g_top, _g_idx, _g_counts, _g_scores):
    scores, idx = ctx.saved_tensors
    score_func, route_norm, route_scale = ctx.cfg
    if g_top is None:
        g_top = torch.zeros(idx.shape, dtype=torch.float32, device=idx.device)
    grad_logits = router_backward(g_top, scores, idx, score_func, route_norm, route_scale)
    return grad_logits, None, None, None, None, None, None, None, None, None, None


router.register_autograd(_router_bwd, setup_context=_router_setup)


# ---------------------------------------------------------------------------
# the gate's backward on bf16 GEMMs: exact three-term split, dW reduction
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::gate_grad_split3", mutates_args=())
def gate_grad_split3(grad_logits: Tensor) -> Tensor:
    """fp32 [N, C] -> bf16 [N, 3C] (hi | mid | lo) with hi + mid + lo == grad_logits."""
    require_gpu(grad_logits)
    d = grad_logits.float().contiguous()
    n, c = d.shape
    out = torch.empty(n, 3 * c, dtype=torch.bfloat16, device=d.device)
    call("moe_gate_grad_split3", ptr(d), n, c, ptr(out), stream_of(d))
    return out


@gate_grad_split3.register_fake
def _(grad_logits):
    n, c = grad_logits.shape
    return grad_logits.new_empty(n, 3 * c, dtype=torch.bfloat16)


@torch.library.custom_op("moe_mi355x::gate_dw_reduce", mutates_args=())
def gate_dw_reduce(partials: Tensor, num_experts: int) -> Tensor:
    """fp32 partials [3E, D] or [2, 3E, D] (token halves) -> bf16 [E, D]:
    bf16((hi + mid) + lo) of the half sums."""
    require_gpu(partials)
    p = partials.float().contiguous()
    parts = 2 if p.dim() == 3 else 1
    d = p.shape[-1]
    if p.shape[-2] != 3 * num_experts or (parts == 2 and p.shape[0] != 2):
        raise ValueError(f"gate_dw_reduce: partials {tuple(p.shape)} for {num_experts} experts")
    out = torch.empty(num_experts, d, dtype=torch.bfloat16, device=p.device)
    call("moe_gate_dw_reduce", ptr(p), parts, num_experts, d, ptr(out), stream_of(p))
    return out


@gate_dw_reduce.register_fake
def _(partials, num_experts):
    return partials.new_empty(num_experts, partials.shape[-1], dtype=torch.bfloat16)


# ---------------------------------------------------------------------------
# shared expert SwiGLU between its GEMMs (feed_forward.py:53-54)
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::swiglu_forward", mutates_args=())
def swiglu_forward(a1: Tensor, a3: Tensor) -> Tensor:
    """h = silu(a1) * a3 with torch's roundings; a1, a3 [..., Hs] bf16 or fp32."""
    require_gpu(a1, a3)
    if a1.shape != a3.shape or a1.dtype != a3.dtype:
        raise ValueError("swiglu_forward: a1 and a3 must have one shape and dtype")
    a1c, a3c = a1.contiguous(), a3.contiguous()
    hs = a1.shape[-1]
    h = torch.empty_like(a1c)
    call("moe_swiglu_fwd", ptr(a1c), ptr(a3c), a1c.numel() // max(hs, 1), hs, _dtype_code(a1c), ptr(h),
         stream_of(a1c))
    return h


@swiglu_forward.register_fake
def _(a1, a3):
    return torch.empty_like(a1)


@torch.library.custom_op("moe_mi355x::swiglu_backward", mutates_args=())
def swiglu_backward(dh: Tensor, a1: Tensor, a3: Tensor) -> Tensor:
    """dgu [rows, 2 Hs]: silu_backward(dh * a3, a1) | dh * silu(a1), torch's roundings."""
    require_gpu(dh, a1, a3)
    if not (dh.shape == a1.shape == a3.shape) or not (dh.dtype == a1.dtype == a3.dtype):
        raise ValueError("swiglu_backward: dh, a1 and a3 must have one shape and dtype")
    hs = a1.shape[-1]
    rows = a1.numel() // max(hs, 1)
    dhc, a1c, a3c = dh.contiguous(), a1.contiguous(), a3.contiguous()
    dgu = torch.empty(rows, 2 * hs, dtype=a1.dtype, device=a1.device)
    call("moe_swiglu_bwd", ptr(dhc), ptr(a1c), ptr(a3c), rows, hs, _dtype_code(a1c), ptr(dgu), stream_of(a1c))
    return dgu


@swiglu_backward.register_fake
def _(dh, a1, a3):
    hs = a1.shape[-1]
    return a1.new_empty(a1.numel() // max(hs, 1), 2 * hs)


# ---------------------------------------------------------------------------
# reorder: counting-sort permutation by expert
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::reorder", mutates_args=())
def reorder(
    top_scores: Tensor, selected_experts: Tensor, num_experts: int
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Returns (scores_sorted [R] f32, token_idx [R] i64, counts [E] i64,
    offsets [E] i32, slot_pos [N,K] i32, tok_pos [N,K] i32)."""
    require_gpu(top_scores, selected_experts)
    idx = selected_experts.contiguous()
    ts = top_scores.float().contiguous()
    n, k = idx.shape
    dev = idx.device
    r = n * k
    scores_sorted = torch.empty(r, dtype=torch.float32, device=dev)
    token_idx = torch.empty(r, dtype=torch.int64, device=dev)
    counts = torch.empty(num_experts, dtype=torch.int64, device=dev)
    offsets = torch.empty(num_experts, dtype=torch.int32, device=dev)
    slot_pos = torch.empty(n, k, dtype=torch.int32, device=dev)
    tok_pos = torch.empty(n, k, dtype=torch.int32, device=dev)
    ws = _workspace(n, num_experts, dev)
    call(
        "moe_reorder", ptr(idx), ptr(ts), n, k, num_experts, ptr(ws), ws.numel(),
                          ptr(scores_sorted), ptr(token_idx), ptr(counts), ptr(offsets),
                          ptr(slot_pos), ptr(tok_pos), stream_of(idx)
    )
    return scores_sorted, token_idx, counts, offsets, slot_pos, tok_pos


@reorder.register_fake
def _(top_scores, selected_experts, num_experts):
    n, k = selected_experts.shape
    e = selected_experts
    return (
        e.new_empty(n * k, dtype=torch.float32),
        e.new_empty(n * k, dtype=torch.int64),
        e.new_empty(num_experts, dtype=torch.int64),
        e.new_empty(num_experts, dtype=torch.int32),
        e.new_empty(n, k, dtype=torch.int32),
        e.new_empty(n, k, dtype=torch.int32),
    )


@torch.library.custom_op("moe_mi355x::reorder_backward", mutates_args=())
def reorder_backward(grad_scores_sorted: Tensor, slot_pos: Tensor) -> Tensor:
    require_gpu(grad_scores_sorted, slot_pos)
    g = grad_scores_sorted.float().contiguous()
    n, k = slot_pos.shape
    out = torch.empty(n, k, dtype=torch.float32, device=g.device)
    call(
        "moe_reorder_bwd", ptr(g), ptr(slot_pos), n, k, ptr(out), stream_of(g)
    )
    return out


@reorder_backward.register_fake
def _(grad_scores_sorted, slot_pos):
    return slot_pos.new_empty(slot_pos.shape, dtype=torch.float32)


def _reorder_setup(ctx, inputs, output):
    _ts, _idx, _e = inputs
    _ss, token_idx, counts, offsets, slot_pos, tok_pos = output
    ctx.save_for_backward(slot_pos)
    ctx.mark_non_differentiable(token_idx, counts, offsets, slot_pos, tok_pos)
    ctx.set_materialize_grads(False)  # no zero-filled grads for the index / saved outputs


def _reorder_bwd(ctx, g_sorted, *_ignored):
    (slot_pos,) = ctx.saved_tensors
    if g_sorted is None:
        return None, None, None
    return reorder_backward(g_sorted, slot_pos), None, None


reorder.register_autograd(_reorder_bwd, setup_context=_reorder_setup)


# ---------------------------------------------------------------------------
# permute: routed_input = x[token_idx] (* score)
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::permute", mutates_args=())
def permute(x: Tensor, slot_pos: Tensor, tok_pos: Tensor, scores_sorted: Tensor | None) -> Tensor:
    require_gpu(x, slot_pos, scores_sorted)
    x = x.contiguous()
    n, d = x.shape
    k = slot_pos.shape[1]
    out = x.new_empty(n * k, d)
    sc = scores_sorted.float().contiguous() if scores_sorted is not None else None
    call(
        "moe_permute", ptr(x), ptr(slot_pos), ptr(sc), n, d, k, _dtype_code(x), ptr(out), stream_of(x)
    )
    return out


@permute.register_fake
def _(x, slot_pos, tok_pos, scores_sorted):
    return x.new_empty(x.shape[0] * slot_pos.shape[1], x.shape[1])


@torch.library.custom_op("moe_mi355x::permute_backward", mutates_args=())
def permute_backward(
    grad_routed: Tensor, x: Tensor, tok_pos: Tensor, scores_sorted: Tensor | None, round_each: bool
) -> tuple[Tensor, Tensor]:
    require_gpu(grad_routed, x, tok_pos, scores_sorted)
    g = grad_routed.contiguous()
    n, d = x.shape
    k = tok_pos.shape[1]
    grad_x = x.new_empty(n, d)
    grad_s = torch.empty(n * k if scores_sorted is not None else 0, dtype=torch.float32, device=x.device)
    sc = scores_sorted.float().contiguous() if scores_sorted is not None else None
    call(
        "moe_permute_bwd", ptr(g), ptr(x), ptr(tok_pos), ptr(sc), n, d, k, _dtype_code(x),
                              int(round_each), ptr(grad_x), ptr(grad_s) if sc is not None else None,
                              stream_of(x)
    )
    return grad_x, grad_s


@permute_backward.register_fake
def _(grad_routed, x, tok_pos, scores_sorted, round_each):
    k = tok_pos.shape[1]
    ns = x.shape[0] * k if scores_sorted is not None else 0
    return x.new_empty(x.shape), x.new_empty(ns, dtype=torch.float32)


def _permute_setup(ctx, inputs, output):
    x, slot_pos, tok_pos, scores_sorted = inputs
    ctx.has_scores = scores_sorted is not None
    ctx.save_for_backward(x, tok_pos, scores_sorted if scores_sorted is not None else None)


def _permute_bwd(ctx, g):
    x, tok_pos, scores_sorted = ctx.saved_tensors
    grad_x, grad_s = permute_backward(g, x, tok_pos, scores_sorted if ctx.has_scores else None,
                                      PERMUTE_BWD_ROUND_EACH)
    return grad_x, None, None, (grad_s if ctx.has_scores else None)


permute.register_autograd(_permute_bwd, setup_context=_permute_setup)


# ---------------------------------------------------------------------------
# grouped SwiGLU experts: _run_experts_grouped_mm
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::grouped_swiglu", mutates_args=())
def grouped_swiglu(
    x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """bf16 grouped SwiGLU. Returns (y [R,D], g [R,H], u [R,H], h [R,H]); g, u, h are
    the saved activations for the backward."""
    require_gpu(x, w1, w2, w3, num_tokens_per_expert)
    for t, name in ((x, "x"), (w1, "w1"), (w2, "w2"), (w3, "w3")):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"grouped_swiglu expects bfloat16 {name}, got {t.dtype}")
    x, w1, w2, w3 = x.contiguous(), w1.contiguous(), w2.contiguous(), w3.contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h_dim, _ = w1.shape
    g = x.new_empty(r, h_dim)
    u = x.new_empty(r, h_dim)
    h = x.new_empty(r, h_dim)
    y = x.new_empty(r, d)
    s = stream_of(x)
    call("moe_grouped_gemm_gate_up", ptr(x), ptr(w1), ptr(w3), ptr(counts), r, e, d, h_dim,
         ptr(g), ptr(u), ptr(h), s)
    call("moe_grouped_gemm_down", ptr(h), ptr(w2), ptr(counts), r, e, d, h_dim, ptr(y), s)
    return y, g, u, h


@grouped_swiglu.register_fake
def _(x, w1, w2, w3, num_tokens_per_expert):
    r, d = x.shape
    h_dim = w1.shape[1]
    return x.new_empty(r, d), x.new_empty(r, h_dim), x.new_empty(r, h_dim), x.new_empty(r, h_dim)


@torch.library.custom_op("moe_mi355x::grouped_swiglu_backward", mutates_args=())
def grouped_swiglu_backward(
    dy: Tensor, x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor,
    g: Tensor, u: Tensor, h: Tensor,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    require_gpu(dy, x, w1, w2, w3, num_tokens_per_expert, g, u, h)
    dy = dy.to(torch.bfloat16).contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h_dim, _ = w1.shape
    dgu = x.new_empty(r, 2 * h_dim)
    dx = x.new_empty(r, d)
    dw1 = torch.empty_like(w1)
    dw2 = torch.empty_like(w2)
    dw3 = torch.empty_like(w3)
    s = stream_of(x)
    call("moe_grouped_gemm_bwd_dgu", ptr(dy), ptr(w2), ptr(g), ptr(u), ptr(counts), r, e, d, h_dim,
         ptr(dgu), s)
    call("moe_grouped_gemm_bwd_dx", ptr(dgu), ptr(w1), ptr(w3), ptr(counts), r, e, d, h_dim, ptr(dx), s)
    call("moe_grouped_gemm_bwd_dw13", ptr(dgu), ptr(x), ptr(counts), r, e, d, h_dim, ptr(dw1),
         ptr(dw3), s)
    call("moe_grouped_gemm_bwd_dw2", ptr(dy), ptr(h), ptr(counts), r, e, d, h_dim, ptr(dw2), s)
    return dx, dw1, dw2, dw3


@grouped_swiglu_backward.register_fake
def _(dy, x, w1, w2, w3, num_tokens_per_expert, g, u, h):
    return x.new_empty(x.shape), torch.empty_like(w1), torch.empty_like(w2), torch.empty_like(w3)


def _gs_setup(ctx, inputs, output):
    x, w1, w2, w3, counts = inputs
    _y, g, u, h = output
    ctx.save_for_backward(x, w1, w2, w3, counts, g, u, h)
    ctx.mark_non_differentiable(g, u, h)
    ctx.set_materialize_grads(False)  # no zero-filled grads for the index / saved outputs


def _gs_bwd(ctx, dy, _dg, _du, _dh):
    x, w1, w2, w3, counts, g, u, h = ctx.saved_tensors
    if dy is None:
        return None, None, None, None, None
    dx, dw1, dw2, dw3 = grouped_swiglu_backward(dy, x, w1, w2, w3, counts, g, u, h)
    return dx, dw1, dw2, dw3, None


grouped_swiglu.register_autograd(_gs_bwd, setup_context=_gs_setup)


# ---------------------------------------------------------------------------
# fp32 grouped SwiGLU experts: _run_experts_for_loop in the input dtype
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::grouped_swiglu_f32", mutates_args=())
def grouped_swiglu_f32(
    x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """fp32 grouped SwiGLU (every product and sum in fp32, as the reference's
    fp32 per-expert matmuls, moe.py:24-50). Returns (y [R,D], g, u, h [R,H]);
    rows past sum(counts) of y are zero."""
    require_gpu(x, w1, w2, w3, num_tokens_per_expert)
    for t, name in ((x, "x"), (w1, "w1"), (w2, "w2"), (w3, "w3")):
        if t.dtype != torch.float32:
            raise TypeError(f"grouped_swiglu_f32 expects float32 {name}, got {t.dtype}")
    x, w1, w2, w3 = x.contiguous(), w1.contiguous(), w2.contiguous(), w3.contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h_dim, _ = w1.shape
    g = x.new_empty(r, h_dim)
    u = x.new_empty(r, h_dim)
    h = x.new_empty(r, h_dim)
    y = x.new_empty(r, d)
    s = stream_of(x)
    call("moe_zero_rows_past_f32", ptr(counts), r, e, ptr(g), h_dim, ptr(u), h_dim, ptr(h), h_dim, ptr(y), d, s)
    call("moe_grouped_gemm_f32_gate_up", ptr(x), ptr(w1), ptr(w3), ptr(counts), r, e, d, h_dim,
         ptr(g), ptr(u), ptr(h), s)
    call("moe_grouped_gemm_f32_down", ptr(h), ptr(w2), ptr(counts), r, e, d, h_dim, ptr(y), s)
    return y, g, u, h


@grouped_swiglu_f32.register_fake
def _(x, w1, w2, w3, num_tokens_per_expert):
    r, d = x.shape
    h_dim = w1.shape[1]
    return x.new_empty(r, d), x.new_empty(r, h_dim), x.new_empty(r, h_dim), x.new_empty(r, h_dim)


@torch.library.custom_op("moe_mi355x::grouped_swiglu_f32_backward", mutates_args=())
def grouped_swiglu_f32_backward(
    dy: Tensor, x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor,
    g: Tensor, u: Tensor, h: Tensor,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    require_gpu(dy, x, w1, w2, w3, num_tokens_per_expert, g, u, h)
    dy = dy.to(torch.float32).contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h_dim, _ = w1.shape
    dg = x.new_empty(r, h_dim)
    du = x.new_empty(r, h_dim)
    dx = x.new_empty(r, d)
    dw1 = torch.empty_like(w1)
    dw2 = torch.empty_like(w2)
    dw3 = torch.empty_like(w3)
    s = stream_of(x)
    call("moe_zero_rows_past_f32", ptr(counts), r, e, ptr(dg), h_dim, ptr(du), h_dim, ptr(dx), d, None, 0, s)
    call("moe_grouped_gemm_f32_bwd_dgu", ptr(dy), ptr(w2), ptr(g), ptr(u), ptr(counts), r, e, d, h_dim,
         ptr(dg), ptr(du), s)
    call("moe_grouped_gemm_f32_bwd_dx", ptr(dg), ptr(du), ptr(w1), ptr(w3), ptr(counts), r, e, d, h_dim,
         ptr(dx), s)
    call("moe_grouped_gemm_f32_bwd_dw_all", ptr(dg), ptr(du), ptr(dy), ptr(x), ptr(h), ptr(counts), r, e, d, h_dim,
         ptr(dw1), ptr(dw3), ptr(dw2), s)
    return dx, dw1, dw2, dw3


@grouped_swiglu_f32_backward.register_fake
def _(dy, x, w1, w2, w3, num_tokens_per_expert, g, u, h):
    return x.new_empty(x.shape), torch.empty_like(w1), torch.empty_like(w2), torch.empty_like(w3)


def _gs32_bwd(ctx, dy, _dg, _du, _dh):
    x, w1, w2, w3, counts, g, u, h = ctx.saved_tensors
    if dy is None:
        return None, None, None, None, None
    dx, dw1, dw2, dw3 = grouped_swiglu_f32_backward(dy, x, w1, w2, w3, counts, g, u, h)
    return dx, dw1, dw2, dw3, None


grouped_swiglu_f32.register_autograd(_gs32_bwd, setup_context=_gs_setup)


# ---------------------------------------------------------------------------
# combine: out = shared + sum of a token's routed rows (deterministic)
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::combine", mutates_args=())
def combine(
    shared_out: Tensor | None, routed_output: Tensor, slot_pos: Tensor, tok_pos: Tensor,
    scores_sorted: Tensor | None,
) -> Tensor:
    require_gpu(shared_out, routed_output, tok_pos, scores_sorted)
    routed = routed_output.contiguous()
    n, k = tok_pos.shape
    d = routed.shape[1]
    base = shared_out.to(routed.dtype).contiguous() if shared_out is not None else None
    out = routed.new_empty(n, d)
    sc = scores_sorted.float().contiguous() if scores_sorted is not None else None
    call(
        "moe_combine", ptr(base), ptr(routed), ptr(tok_pos), ptr(sc), n, d, k, _dtype_code(routed),
                          ptr(out), stream_of(routed)
    )
    return out


@combine.register_fake
def _(shared_out, routed_output, slot_pos, tok_pos, scores_sorted):
    return routed_output.new_empty(tok_pos.shape[0], routed_output.shape[1])


@torch.library.custom_op("moe_mi355x::combine_backward", mutates_args=())
def combine_backward(
    grad_out: Tensor, routed_output: Tensor, slot_pos: Tensor, tok_pos: Tensor,
    scores_sorted: Tensor | None,
) -> tuple[Tensor, Tensor]:
    require_gpu(grad_out, routed_output, slot_pos, tok_pos, scores_sorted)
    g = grad_out.to(routed_output.dtype).contiguous()
    n, k = tok_pos.shape
    d = g.shape[1]
    grad_routed = g.new_empty(n * k, d)
    grad_s = torch.empty(n * k if scores_sorted is not None else 0, dtype=torch.float32, device=g.device)
    sc = scores_sorted.float().contiguous() if scores_sorted is not None else None
    call(
        "moe_combine_bwd", ptr(g), ptr(routed_output), ptr(slot_pos), ptr(tok_pos), ptr(sc), n, d, k,
                              _dtype_code(g), ptr(grad_routed), ptr(grad_s) if sc is not None else None,
                              stream_of(g)
    )
    return grad_routed, grad_s


@combine_backward.register_fake
def _(grad_out, routed_output, slot_pos, tok_pos, scores_sorted):
    n, k = tok_pos.shape
    ns = n * k if scores_sorted is not None else 0
    return routed_output.new_empty(n * k, routed_output.shape[1]), grad_out.new_empty(ns, dtype=torch.float32)


def _combine_setup(ctx, inputs, output):
    shared_out, routed_output, slot_pos, tok_pos, scores_sorted = inputs
    ctx.has_shared = shared_out is not None
    ctx.shared_dtype = shared_out.dtype if shared_out is not None else None
    ctx.has_scores = scores_sorted is not None
    ctx.save_for_backward(routed_output if ctx.has_scores else None, slot_pos, tok_pos, scores_sorted)


def _combine_bwd(ctx, g):
    routed, slot_pos, tok_pos, scores_sorted = ctx.saved_tensors
    if ctx.has_scores:
        grad_routed, grad_s = combine_backward(g, routed, slot_pos, tok_pos, scores_sorted)
    else:
        dummy = g.new_empty(0, g.shape[1])
        grad_routed, _ = combine_backward(g, dummy, slot_pos, tok_pos, None)
        grad_s = None
    grad_shared = g.to(ctx.shared_dtype) if ctx.has_shared else None
    return grad_shared, grad_routed, None, None, grad_s


combine.register_autograd(_combine_bwd, setup_context=_combine_setup)


# ---------------------------------------------------------------------------
# gpt-oss experts: biased, clamped SwiGLU with interleaved mlp1 rows
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::grouped_swiglu_oss", mutates_args=())
def grouped_swiglu_oss(
    x: Tensor, mlp1_weight: Tensor, mlp1_bias: Tensor, mlp2_weight: Tensor, mlp2_bias: Tensor,
    num_tokens_per_expert: Tensor, swiglu_limit: float,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """gpt-oss grouped experts (gpt_oss/moe.py:92-122) in bf16: returns y [R, D]
    and the saved g, u (biased pre-clamp halves of h1) and h [R, H]."""
    require_gpu(x, mlp1_weight, mlp1_bias, mlp2_weight, mlp2_bias, num_tokens_per_expert)
    x, w1, w2 = (t.contiguous() for t in (x, mlp1_weight, mlp2_weight))
    for t, name in ((x, "x"), (w1, "mlp1_weight"), (w2, "mlp2_weight")):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"grouped_swiglu_oss expects bfloat16 {name}, got {t.dtype}")
    b1 = mlp1_bias.to(torch.bfloat16).contiguous()
    b2 = mlp2_bias.to(torch.bfloat16).contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h2, _ = w1.shape
    h_dim = h2 // 2
    s = stream_of(x)
    g = x.new_empty(r, h_dim)
    u = x.new_empty(r, h_dim)
    h = x.new_empty(r, h_dim)
    y = x.new_empty(r, d)
    call("moe_grouped_gemm_oss_gate_up", ptr(x), ptr(w1), ptr(b1), ptr(counts), r, e, d, h_dim, float(swiglu_limit),
         ptr(g), ptr(u), ptr(h), s)
    call("moe_grouped_gemm_oss_down", ptr(h), ptr(w2), ptr(b2), ptr(counts), r, e, d, h_dim, ptr(y), s)
    return y, g, u, h


@grouped_swiglu_oss.register_fake
def _(x, mlp1_weight, mlp1_bias, mlp2_weight, mlp2_bias, num_tokens_per_expert, swiglu_limit):
    r, d = x.shape
    h_dim = mlp1_weight.shape[1] // 2
    return x.new_empty(r, d), x.new_empty(r, h_dim), x.new_empty(r, h_dim), x.new_empty(r, h_dim)


@torch.library.custom_op("moe_mi355x::grouped_swiglu_oss_backward", mutates_args=())
def grouped_swiglu_oss_backward(
    dy: Tensor, x: Tensor, mlp1_weight: Tensor, mlp1_bias: Tensor, mlp2_weight: Tensor, mlp2_bias: Tensor,
    num_tokens_per_expert: Tensor, g: Tensor, u: Tensor, h: Tensor, swiglu_limit: float,
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Gradients (dx, dmlp1_weight, dmlp1_bias, dmlp2_weight, dmlp2_bias); the
    bias gradients are fp32 per-expert sums in a fixed order, cast to the bias dtype."""
    require_gpu(dy, x, mlp1_weight, mlp2_weight, num_tokens_per_expert, g, u, h)
    dy = dy.to(torch.bfloat16).contiguous()
    x, w1, w2 = (t.contiguous() for t in (x, mlp1_weight, mlp2_weight))
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h2, _ = w1.shape
    h_dim = h2 // 2
    s = stream_of(x)
    dgu = x.new_empty(r, 2 * h_dim)
    call("moe_grouped_gemm_oss_bwd_dgu", ptr(dy), ptr(w2), ptr(g), ptr(u), ptr(counts), r, e, d, h_dim,
         float(swiglu_limit), ptr(dgu), s)
    dx = x.new_empty(r, d)
    call("moe_grouped_gemm_oss_bwd_dx", ptr(dgu), ptr(w1), ptr(counts), r, e, d, h_dim, ptr(dx), s)
    dw1 = torch.empty_like(w1)
    call("moe_grouped_gemm_oss_bwd_dw1", ptr(dgu), ptr(x), ptr(counts), r, e, d, h_dim, ptr(dw1), s)
    dw2 = torch.empty_like(w2)
    call("moe_grouped_gemm_bwd_dw2", ptr(dy), ptr(h), ptr(counts), r, e, d, h_dim, ptr(dw2), s)
    db1 = torch.empty(e, 2 * h_dim, dtype=torch.float32, device=x.device)
    call("moe_grouped_col_sum", ptr(dgu), 2 * h_dim, ptr(counts), r, e, h_dim, ptr(db1), 2 * h_dim, 2, s)
    call("moe_grouped_col_sum", dgu.data_ptr() + 2 * h_dim, 2 * h_dim, ptr(counts), r, e, h_dim,
         db1.data_ptr() + 4, 2 * h_dim, 2, s)
    db2 = torch.empty(e, d, dtype=torch.float32, device=x.device)
    call("moe_grouped_col_sum", ptr(dy), d, ptr(counts), r, e, d, ptr(db2), d, 1, s)
    return dx, dw1, db1.to(mlp1_bias.dtype), dw2, db2.to(mlp2_bias.dtype)


@grouped_swiglu_oss_backward.register_fake
def _(dy, x, mlp1_weight, mlp1_bias, mlp2_weight, mlp2_bias, num_tokens_per_expert, g, u, h, swiglu_limit):
    return (x.new_empty(x.shape), torch.empty_like(mlp1_weight), torch.empty_like(mlp1_bias),
            torch.empty_like(mlp2_weight), torch.empty_like(mlp2_bias))


def _oss_setup(ctx, inputs, output):
    x, w1, b1, w2, b2, counts, limit = inputs
    _, g, u, h = output
    ctx.save_for_backward(x, w1, b1, w2, b2, counts, g, u, h)
    ctx.swiglu_limit = limit
    ctx.set_materialize_grads(False)


def _oss_bwd(ctx, dy, _dg, _du, _dh):
    x, w1, b1, w2, b2, counts, g, u, h = ctx.saved_tensors
    if dy is None:
        return None, None, None, None, None, None, None
    dx, dw1, db1, dw2, db2 = grouped_swiglu_oss_backward(dy, x, w1, b1, w2, b2, counts, g, u, h, ctx.swiglu_limit)
    return dx, dw1, db1, dw2, db2, None, None


grouped_swiglu_oss.register_autograd(_oss_bwd, setup_context=_oss_setup)


# ---------------------------------------------------------------------------
# fp8 e4m3 grouped SwiGLU experts (dynamic rowwise scaling, fp32 accumulate)
# ---------------------------------------------------------------------------
FP8 = torch.uint8  # fp8 e4m3fn bytes as produced by the quantizers


def _quant_rows(x: Tensor, cols: int) -> tuple[Tensor, Tensor]:
    """x viewed as [rows, cols] bf16 -> (q uint8 [rows, cols], scale f32 [rows])."""
    rows = x.numel() // cols
    q = torch.empty(rows, cols, dtype=FP8, device=x.device)
    s = torch.empty(rows, dtype=torch.float32, device=x.device)
    call("moe_fp8_quant_rows", ptr(x), rows, cols, ptr(q), ptr(s), stream_of(x))
    return q, s


# widest rows the row quantizers with a column amax on the side take (their
# rows stay in registers)
AMAX_SIDE_MAX_COLS = 8192


def _amax_shape(e: int, cols: int) -> tuple[int, ...]:
    """Shape of a column amax taken on the side of a row quantization: [E, cols],
    or empty when the rows are too wide (the transposed quantizer then takes its
    own amax pass)."""
    return (e, cols) if cols <= AMAX_SIDE_MAX_COLS else (0,)


def _quant_rows_colamax(w: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """w [E, A, B] bf16 -> (q [E, A, B] fp8 with a scale per row, scale [E * A],
    column amax [E, B] over A): the row quantization and, on the side, what the
    transposed one needs, from one read."""
    e, a, b = w.shape
    if b > AMAX_SIDE_MAX_COLS:
        q, s = _quant_rows(w, b)
        return q.view(e, a, b), s, w.new_empty(0, dtype=torch.float32)
    q = torch.empty(e, a, b, dtype=FP8, device=w.device)
    s = torch.empty(e * a, dtype=torch.float32, device=w.device)
    amax = torch.zeros(e, b, dtype=torch.float32, device=w.device)
    call("moe_fp8_quant_rows_colamax", ptr(w), e, a, b, ptr(q), ptr(s), ptr(amax), stream_of(w))
    return q, s, amax


def _quant_rows_groupamax(x: Tensor, counts: Tensor, e: int, pieces: int = 1) -> tuple[Tensor, Tensor, Tensor]:
    """x [R, C] bf16 in expert token groups -> (q [R, C] fp8 with a scale per row
    piece of C / pieces columns, scale [R * pieces], the column amax [E, C] of
    each group): the row quantization and, on the side, what the token-transposed
    one needs, from one read."""
    r, c = x.shape
    if c > AMAX_SIDE_MAX_COLS:
        q, sc = _quant_rows(x, c // pieces)
        return q.view(r, c), sc, x.new_empty(0, dtype=torch.float32)
    q = torch.empty(r, c, dtype=FP8, device=x.device)
    sc = torch.empty(r * pieces, dtype=torch.float32, device=x.device)
    amax = torch.zeros(e, c, dtype=torch.float32, device=x.device)
    call("moe_fp8_quant_rows_groupamax", ptr(x), ptr(counts), r, e, c, pieces, ptr(q), ptr(sc), ptr(amax),
         stream_of(x))
    return q, sc, amax


def _quant_cols_t(w: Tensor, amax: Tensor, q: Tensor, q_offset: int, q_estride: int, q_ld: int, scale: Tensor,
                  s_offset: int, s_estride: int) -> None:
    """Per expert and column of w [E, A, B]: the scale of the column amax and the
    column quantized as a row of q (transposed); from the known amax when there
    is one (one read of w), else with its own amax pass."""
    e, a, b = w.shape
    qp, sp = q.data_ptr() + q_offset, scale.data_ptr() + 4 * s_offset
    if amax.numel():
        call("moe_fp8_quant_cols_t_amax", ptr(w), ptr(amax), e, a, b, qp, q_estride, q_ld, sp, s_estride,
             stream_of(w))
    else:
        call("moe_fp8_quant_cols_t", ptr(w), e, a, b, qp, q_estride, q_ld, sp, s_estride, stream_of(w))


def _padded_rows(r: int, e: int) -> int:
    """Width of the token-transposed layout (token groups 128-aligned): a multiple
    of 128, so that every row and every group in it starts on a 128-byte line."""
    n = lib().moe_fp8_padded_rows(r, e)
    return (n + 127) // 128 * 128


def _quant_tokens_t(x: Tensor, counts: Tensor, e: int, rpad: int,
                    amax: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """x [R, C] bf16 in expert token groups -> (q [C, rpad], scale [E, C]); from
    the groups' known column amax when there is one (one read of x), else with
    its own amax pass."""
    r, c = x.shape
    q = torch.empty(c, rpad, dtype=FP8, device=x.device)
    s = torch.empty(e, c, dtype=torch.float32, device=x.device)
    if amax is not None and amax.numel():
        call("moe_fp8_quant_tokens_t_amax", ptr(x), ptr(amax), ptr(counts), r, e, c, rpad, ptr(q), ptr(s),
             stream_of(x))
    else:
        call("moe_fp8_quant_tokens_t", ptr(x), ptr(counts), r, e, c, rpad, ptr(q), ptr(s), stream_of(x))
    return q, s


@torch.library.custom_op("moe_mi355x::grouped_swiglu_fp8", mutates_args=())
def grouped_swiglu_fp8(
    x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """fp8 e4m3 grouped SwiGLU: x, h quantized per token row, weights per
    output row; fp32 accumulate; bf16 outputs (y, g, u, h), then the column
    amax the backward's transposed quantizations use, taken on the side of the
    forward's: the weights' over their output rows (w1, w3 [E, D], w2 [E, H])
    and x's and h's over each expert's tokens ([E, D], [E, H])."""
    require_gpu(x, w1, w2, w3, num_tokens_per_expert)
    for t, name in ((x, "x"), (w1, "w1"), (w2, "w2"), (w3, "w3")):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"grouped_swiglu_fp8 expects bfloat16 {name}, got {t.dtype}")
    x, w1, w2, w3 = x.contiguous(), w1.contiguous(), w2.contiguous(), w3.contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    qx, sx, amx = _quant_rows_groupamax(x, counts, w1.shape[0])
    y, g, u, h, am1, am3, am2, amh = _fp8_experts_forward(qx, sx, w1, w2, w3, counts)
    return y, g, u, h, am1, am3, am2, amx, amh


def _fp8_experts_forward(qx: Tensor, sx: Tensor, w1: Tensor, w2: Tensor, w3: Tensor,
                         counts: Tensor) -> tuple[Tensor, ...]:
    """grouped_swiglu_fp8 from the row-quantized routed rows (qx, sx): the weights'
    quantizations, gate_up, h's quantization, down. Returns (y, g, u, h, amax_w1,
    amax_w3, amax_w2, amax_h)."""
    r, d = qx.shape
    e, h_dim, _ = w1.shape
    s = stream_of(w1)
    qw1, sw1, am1 = _quant_rows_colamax(w1)
    qw3, sw3, am3 = _quant_rows_colamax(w3)
    qw2, sw2, am2 = _quant_rows_colamax(w2)
    g = w1.new_empty(r, h_dim)
    u = w1.new_empty(r, h_dim)
    h = w1.new_empty(r, h_dim)
    y = w1.new_empty(r, d)
    call("moe_fp8_gemm_gate_up", ptr(qx), ptr(sx), ptr(qw1), ptr(sw1), ptr(qw3), ptr(sw3), ptr(counts), r, e, d,
         h_dim, ptr(g), ptr(u), ptr(h), s)
    qh, sh, amh = _quant_rows_groupamax(h, counts, e)
    call("moe_fp8_gemm_down", ptr(qh), ptr(sh), ptr(qw2), ptr(sw2), ptr(counts), r, e, d, h_dim, ptr(y), s)
    return y, g, u, h, am1, am3, am2, amh


@grouped_swiglu_fp8.register_fake
def _(x, w1, w2, w3, num_tokens_per_expert):
    r, d = x.shape
    e, h_dim = w1.shape[0], w1.shape[1]
    f32 = lambda *shape: x.new_empty(*shape, dtype=torch.float32)  # noqa: E731
    return (x.new_empty(r, d), x.new_empty(r, h_dim), x.new_empty(r, h_dim), x.new_empty(r, h_dim),
            f32(*_amax_shape(e, d)), f32(*_amax_shape(e, d)), f32(*_amax_shape(e, h_dim)),
            f32(*_amax_shape(e, d)), f32(*_amax_shape(e, h_dim)))


@torch.library.custom_op("moe_mi355x::grouped_swiglu_fp8_backward", mutates_args=())
def grouped_swiglu_fp8_backward(
    dy: Tensor, x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor,
    g: Tensor, u: Tensor, h: Tensor, amax_w1: Tensor, amax_w3: Tensor, amax_w2: Tensor, amax_x: Tensor,
    amax_h: Tensor,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients of grouped_swiglu_fp8. amax_* are the forward's column amax of
    the weights and of x and h per token group (empty tensors: the transposed
    quantizers take their own)."""
    require_gpu(dy, x, w1, w2, w3, num_tokens_per_expert, g, u, h)
    dy = dy.to(torch.bfloat16).contiguous()
    x = x.contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    e = w1.shape[0]
    qdy, sdy, amdy = _quant_rows_groupamax(dy, counts, e)
    return _fp8_experts_backward(
        qdy, sdy, w1, w2, w3, counts, g, u, h, amax_w1, amax_w3, amax_w2, amax_h,
        lambda rpad: _quant_tokens_t(x, counts, e, rpad, amax_x),
        lambda rpad: _quant_tokens_t(dy, counts, e, rpad, amdy))


def _fp8_experts_backward(qdy: Tensor, sdy: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, counts: Tensor, g: Tensor,
                          u: Tensor, h: Tensor, amax_w1: Tensor, amax_w3: Tensor, amax_w2: Tensor, amax_h: Tensor,
                          x_tokens_t, dy_tokens_t) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """grouped_swiglu_fp8_backward from the row-quantized output gradient (qdy,
    sdy); x_tokens_t(rpad) and dy_tokens_t(rpad) give the token-transposed layouts
    of the routed x and dy. Returns (dx, dw1, dw2, dw3)."""
    r, d = qdy.shape
    e, h_dim, _ = w1.shape
    dev = w1.device
    s = stream_of(w1)
    # dh = dy . w2 (contraction over D): dy per row, w2 per (e, h) column over D
    qw2t = torch.empty(e, h_dim, d, dtype=FP8, device=dev)
    sw2t = torch.empty(e, h_dim, dtype=torch.float32, device=dev)
    _quant_cols_t(w2.contiguous(), amax_w2.contiguous(), qw2t, 0, h_dim * d, d, sw2t, 0, h_dim)
    dgu = w1.new_empty(r, 2 * h_dim)
    call("moe_fp8_gemm_bwd_dgu", ptr(qdy), ptr(sdy), ptr(qw2t), ptr(sw2t), ptr(g), ptr(u), ptr(counts), r, e, d,
         h_dim, ptr(dgu), s)
    # dx = dg . w1 + du . w3 (contraction over H): one scale per dg / du row half,
    # w1 and w3 per (e, d) column over H, written side by side as [E, D, 2H]
    qdgu, sdgu, amdgu = _quant_rows_groupamax(dgu, counts, e, pieces=2)
    qw13t = torch.empty(e, d, 2 * h_dim, dtype=FP8, device=dev)
    sw13t = torch.empty(e, 2, d, dtype=torch.float32, device=dev)
    _quant_cols_t(w1.contiguous(), amax_w1.contiguous(), qw13t, 0, d * 2 * h_dim, 2 * h_dim, sw13t, 0, 2 * d)
    _quant_cols_t(w3.contiguous(), amax_w3.contiguous(), qw13t, h_dim, d * 2 * h_dim, 2 * h_dim, sw13t, d, 2 * d)
    dx = w1.new_empty(r, d)
    call("moe_fp8_gemm_bwd_dx", ptr(qdgu), ptr(sdgu), ptr(qw13t), ptr(sw13t), ptr(counts), r, e, d, h_dim,
         ptr(dx), s)
    # weight gradients: contraction over each expert's tokens (per-group scales)
    rpad = _padded_rows(r, e)
    qdgut, sdgut = _quant_tokens_t(dgu, counts, e, rpad, amdgu)
    qxt, sxt = x_tokens_t(rpad)
    dw1 = torch.empty_like(w1)
    dw3 = torch.empty_like(w3)
    call("moe_fp8_gemm_bwd_dw13", ptr(qdgut), ptr(sdgut), ptr(qxt), ptr(sxt), ptr(counts), r, rpad, e, d, h_dim,
         ptr(dw1), ptr(dw3), s)
    qdyt, sdyt = dy_tokens_t(rpad)
    qht, sht = _quant_tokens_t(h, counts, e, rpad, amax_h)
    dw2 = torch.empty_like(w2)
    call("moe_fp8_gemm_bwd_dw2", ptr(qdyt), ptr(sdyt), ptr(qht), ptr(sht), ptr(counts), r, rpad, e, d, h_dim,
         ptr(dw2), s)
    return dx, dw1, dw2, dw3


@grouped_swiglu_fp8_backward.register_fake
def _(dy, x, w1, w2, w3, num_tokens_per_expert, g, u, h, amax_w1, amax_w3, amax_w2, amax_x, amax_h):
    return x.new_empty(x.shape), torch.empty_like(w1), torch.empty_like(w2), torch.empty_like(w3)


def _gs8_setup(ctx, inputs, output):
    x, w1, w2, w3, counts = inputs
    _y, g, u, h, *amax = output
    ctx.save_for_backward(x, w1, w2, w3, counts, g, u, h, *amax)
    ctx.mark_non_differentiable(g, u, h, *amax)
    ctx.set_materialize_grads(False)


def _gs8_bwd(ctx, dy, *_unused):
    x, w1, w2, w3, counts, g, u, h, *amax = ctx.saved_tensors
    if dy is None:
        return None, None, None, None, None
    dx, dw1, dw2, dw3 = grouped_swiglu_fp8_backward(dy, x, w1, w2, w3, counts, g, u, h, *amax)
    return dx, dw1, dw2, dw3, None


grouped_swiglu_fp8.register_autograd(_gs8_bwd, setup_context=_gs8_setup)


# ---------------------------------------------------------------------------
# MXFP8 grouped SwiGLU experts (e8m0 scales per 32 elements along the
# contraction, RCEIL; fp32 accumulate)
# ---------------------------------------------------------------------------
MX_BLOCK = 32


def _mx_quant_rows(x: Tensor, cols: int) -> tuple[Tensor, Tensor]:
    """x viewed as [rows, cols] bf16 -> (q uint8 [rows, cols], e8m0 uint8 [rows, cols / 32])."""
    rows = x.numel() // cols
    q = torch.empty(rows, cols, dtype=FP8, device=x.device)
    s = torch.empty(rows, cols // MX_BLOCK, dtype=torch.uint8, device=x.device)
    call("moe_mxfp8_quant_rows", ptr(x), rows, cols, ptr(q), ptr(s), stream_of(x))
    return q, s


def _mx_padded_rows(r: int, e: int) -> int:
    """As _padded_rows: r + 127 e rounded up to 128 (token groups 128-aligned)."""
    return (int(lib().moe_mxfp8_padded_rows(r, e)) + 127) // 128 * 128


def _mx_quant_tokens_t(x: Tensor, counts: Tensor, e: int, rpad: int) -> tuple[Tensor, Tensor]:
    """x [R, C] bf16 in expert token groups -> (q [C, rpad], e8m0 [rpad / 32, C])."""
    r, c = x.shape
    q = torch.empty(c, rpad, dtype=FP8, device=x.device)
    s = torch.empty(rpad // MX_BLOCK, c, dtype=torch.uint8, device=x.device)
    call("moe_mxfp8_quant_tokens_t", ptr(x), ptr(counts), r, e, c, rpad, ptr(q), ptr(s), stream_of(x))
    return q, s


def _check_bf16(op: str, **tensors: Tensor) -> None:
    for name, t in tensors.items():
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{op} expects bfloat16 {name}, got {t.dtype}")


def _mx_dual_tokens(x: Tensor, counts: Tensor, e: int, rpad: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """One read of x [R, C] (token groups) -> the row-wise MX layout (q [R, C],
    e8m0 [R, C / 32]) and the token-transposed one (q [C, rpad], e8m0 [rpad / 32, C])."""
    r, c = x.shape
    qr = torch.empty(r, c, dtype=FP8, device=x.device)
    sr = torch.empty(r, c // MX_BLOCK, dtype=torch.uint8, device=x.device)
    qt = torch.empty(c, rpad, dtype=FP8, device=x.device)
    st = torch.empty(rpad // MX_BLOCK, c, dtype=torch.uint8, device=x.device)
    call("moe_mxfp8_quant_dual_tokens", ptr(x), ptr(counts), r, e, c, rpad, ptr(qr), ptr(sr), ptr(qt), ptr(st),
         stream_of(x))
    return qr, sr, qt, st


def _mx_weights(w1: Tensor, w2: Tensor, w3: Tensor, transposed: bool) -> tuple[Tensor, ...]:
    """Row-wise MX layouts of w1, w3 (blocks along D) and w2 (along H); with
    `transposed`, the same reads also write the backward's layouts: w2^T
    [E, H, D] (blocks along D) and [w1^T | w3^T] [E, D, 2H] (blocks along H)."""
    e, h_dim, d = w1.shape
    dev = w1.device
    s = stream_of(w1)
    if not transposed:
        qw1, sw1 = _mx_quant_rows(w1, d)
        qw3, sw3 = _mx_quant_rows(w3, d)
        qw2, sw2 = _mx_quant_rows(w2, h_dim)
        return qw1, sw1, qw3, sw3, qw2, sw2
    qw1 = torch.empty(e * h_dim, d, dtype=FP8, device=dev)
    sw1 = torch.empty(e * h_dim, d // MX_BLOCK, dtype=torch.uint8, device=dev)
    qw3, sw3 = torch.empty_like(qw1), torch.empty_like(sw1)
    qw2 = torch.empty(e * d, h_dim, dtype=FP8, device=dev)
    sw2 = torch.empty(e * d, h_dim // MX_BLOCK, dtype=torch.uint8, device=dev)
    qw2t = torch.empty(e, h_dim, d, dtype=FP8, device=dev)
    sw2t = torch.empty(e, h_dim, d // MX_BLOCK, dtype=torch.uint8, device=dev)
    nb = 2 * h_dim // MX_BLOCK
    qw13t = torch.empty(e, d, 2 * h_dim, dtype=FP8, device=dev)
    sw13t = torch.empty(e, d, nb, dtype=torch.uint8, device=dev)
    call("moe_mxfp8_quant_dual_cols", ptr(w2), e, d, h_dim, ptr(qw2), ptr(sw2), ptr(qw2t), h_dim * d, d, ptr(sw2t),
         h_dim * (d // MX_BLOCK), d // MX_BLOCK, s)
    call("moe_mxfp8_quant_dual_cols", ptr(w1), e, h_dim, d, ptr(qw1), ptr(sw1), ptr(qw13t), d * 2 * h_dim, 2 * h_dim,
         ptr(sw13t), d * nb, nb, s)
    call("moe_mxfp8_quant_dual_cols", ptr(w3), e, h_dim, d, ptr(qw3), ptr(sw3), qw13t.data_ptr() + h_dim,
         d * 2 * h_dim, 2 * h_dim, sw13t.data_ptr() + h_dim // MX_BLOCK, d * nb, nb, s)
    return qw1, sw1, qw3, sw3, qw2, sw2, qw2t, sw2t, qw13t, sw13t


@torch.library.custom_op("moe_mi355x::grouped_swiglu_mxfp8", mutates_args=())
def grouped_swiglu_mxfp8(
    x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor, for_backward: bool = False
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """MXFP8 grouped SwiGLU: x, h and the weights quantized in 32-element
    blocks along each GEMM's contraction; bf16 outputs (y, g, u, h). With
    `for_backward`, the same quantizer reads also produce the layouts the
    backward contracts over (x^T, h^T per token group; w1^T, w3^T, w2^T),
    returned after (y, g, u, h); otherwise those are empty."""
    require_gpu(x, w1, w2, w3, num_tokens_per_expert)
    _check_bf16("grouped_swiglu_mxfp8", x=x, w1=w1, w2=w2, w3=w3)
    x, w1, w2, w3 = x.contiguous(), w1.contiguous(), w2.contiguous(), w3.contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h_dim, _ = w1.shape
    s = stream_of(x)
    def empty():  # distinct placeholders: custom-op outputs may not alias each other
        return x.new_empty(0, dtype=torch.uint8)
    if for_backward:
        rpad = _mx_padded_rows(r, e)
        qx, sx, qxt, sxt = _mx_dual_tokens(x, counts, e, rpad)
        qw1, sw1, qw3, sw3, qw2, sw2, qw2t, sw2t, qw13t, sw13t = _mx_weights(w1, w2, w3, True)
    else:
        qx, sx = _mx_quant_rows(x, d)
        qw1, sw1, qw3, sw3, qw2, sw2 = _mx_weights(w1, w2, w3, False)
        qxt, sxt, qw2t, sw2t, qw13t, sw13t = (empty() for _ in range(6))
    g = x.new_empty(r, h_dim)
    u = x.new_empty(r, h_dim)
    h = x.new_empty(r, h_dim)
    y = x.new_empty(r, d)
    call("moe_mxfp8_gemm_gate_up", ptr(qx), ptr(sx), ptr(qw1), ptr(sw1), ptr(qw3), ptr(sw3), ptr(counts), r, e, d,
         h_dim, ptr(g), ptr(u), ptr(h), s)
    if for_backward:
        qh, sh, qht, sht = _mx_dual_tokens(h, counts, e, rpad)
    else:
        qh, sh = _mx_quant_rows(h, h_dim)
        qht, sht = empty(), empty()
    call("moe_mxfp8_gemm_down", ptr(qh), ptr(sh), ptr(qw2), ptr(sw2), ptr(counts), r, e, d, h_dim, ptr(y), s)
    return y, g, u, h, qxt, sxt, qht, sht, qw2t, sw2t, qw13t, sw13t


@grouped_swiglu_mxfp8.register_fake
def _(x, w1, w2, w3, num_tokens_per_expert, for_backward=False):
    r, d = x.shape
    e, h_dim, _ = w1.shape
    bf = (x.new_empty(r, d), x.new_empty(r, h_dim), x.new_empty(r, h_dim), x.new_empty(r, h_dim))
    u8 = lambda *shape: x.new_empty(*shape, dtype=torch.uint8)  # noqa: E731
    if not for_backward:
        return (*bf, *(u8(0) for _ in range(8)))
    rpad = (r + e * 127 + 127) // 128 * 128  # _mx_padded_rows
    return (*bf, u8(d, rpad), u8(rpad // 32, d), u8(h_dim, rpad), u8(rpad // 32, h_dim),
            u8(e, h_dim, d), u8(e, h_dim, d // 32), u8(e, d, 2 * h_dim), u8(e, d, 2 * h_dim // 32))


@torch.library.custom_op("moe_mi355x::grouped_swiglu_mxfp8_backward", mutates_args=())
def grouped_swiglu_mxfp8_backward(
    dy: Tensor, x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor,
    g: Tensor, u: Tensor, h: Tensor, qxt: Tensor, sxt: Tensor, qht: Tensor, sht: Tensor,
    qw2t: Tensor, sw2t: Tensor, qw13t: Tensor, sw13t: Tensor,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients from the forward's transposed quantizations; dy and dgu are
    quantized once each, in both layouts."""
    require_gpu(dy, x, w1, w2, w3, num_tokens_per_expert, g, u, h)
    dy = dy.to(torch.bfloat16).contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h_dim, _ = w1.shape
    s = stream_of(x)
    rpad = _mx_padded_rows(r, e)
    if qxt.numel() == 0:  # the forward ran without for_backward
        qxt, sxt = _mx_quant_tokens_t(x.contiguous(), counts, e, rpad)
        qht, sht = _mx_quant_tokens_t(h, counts, e, rpad)
        *_, qw2t, sw2t, qw13t, sw13t = _mx_weights(w1.contiguous(), w2.contiguous(), w3.contiguous(), True)
    # dh = dy . w2 (contraction over D)
    qdy = _mx_dual_tokens(dy, counts, e, rpad)
    return _mx_experts_backward(qdy, r, d, w1, w2, w3, counts, g, u, h, qxt, sxt, qht, sht, qw2t, sw2t, qw13t,
                                sw13t, rpad)


def _mx_experts_backward(qdy, r, d, w1, w2, w3, counts, g, u, h, qxt, sxt, qht, sht, qw2t, sw2t, qw13t, sw13t, rpad):
    """dx (routed rows), dw1, dw2, dw3 of the MXFP8 experts from dy's two MX
    layouts (qdy = (q rows, e8m0 rows, q tokens^T, e8m0 tokens^T))."""
    qdy, sdy, qdyt, sdyt = qdy
    e, h_dim, _ = w1.shape
    s = stream_of(g)
    dgu = g.new_empty(r, 2 * h_dim)
    call("moe_mxfp8_gemm_bwd_dgu", ptr(qdy), ptr(sdy), ptr(qw2t), ptr(sw2t), ptr(g), ptr(u), ptr(counts), r, e, d,
         h_dim, ptr(dgu), s)
    # dx = dg . w1 + du . w3 (contraction over H; blocks never straddle the halves)
    qdgu, sdgu, qdgut, sdgut = _mx_dual_tokens(dgu, counts, e, rpad)
    dx = g.new_empty(r, d)
    call("moe_mxfp8_gemm_bwd_dx", ptr(qdgu), ptr(sdgu), ptr(qw13t), ptr(sw13t), ptr(counts), r, e, d, h_dim,
         ptr(dx), s)
    # weight gradients: contraction over each expert's tokens (groups padded to 32)
    dw1 = torch.empty_like(w1)
    dw3 = torch.empty_like(w3)
    call("moe_mxfp8_gemm_bwd_dw13", ptr(qdgut), ptr(sdgut), ptr(qxt), ptr(sxt), ptr(counts), r, rpad, e, d, h_dim,
         ptr(dw1), ptr(dw3), s)
    dw2 = torch.empty_like(w2)
    call("moe_mxfp8_gemm_bwd_dw2", ptr(qdyt), ptr(sdyt), ptr(qht), ptr(sht), ptr(counts), r, rpad, e, d, h_dim,
         ptr(dw2), s)
    return dx, dw1, dw2, dw3


@grouped_swiglu_mxfp8_backward.register_fake
def _(dy, x, w1, w2, w3, num_tokens_per_expert, g, u, h, *quantized):
    return x.new_empty(x.shape), torch.empty_like(w1), torch.empty_like(w2), torch.empty_like(w3)


def _gsmx_setup(ctx, inputs, output):
    x, w1, w2, w3, counts, _for_backward = inputs
    _y, g, u, h, *quantized = output
    ctx.save_for_backward(x, w1, w2, w3, counts, g, u, h, *quantized)
    ctx.mark_non_differentiable(g, u, h, *quantized)
    ctx.set_materialize_grads(False)


def _gsmx_bwd(ctx, dy, *_unused):
    x, w1, w2, w3, counts, g, u, h, *quantized = ctx.saved_tensors
    if dy is None:
        return None, None, None, None, None, None
    dx, dw1, dw2, dw3 = grouped_swiglu_mxfp8_backward(dy, x, w1, w2, w3, counts, g, u, h, *quantized)
    return dx, dw1, dw2, dw3, None, None


grouped_swiglu_mxfp8.register_autograd(_gsmx_bwd, setup_context=_gsmx_setup)


# ---------------------------------------------------------------------------
# bf16 grouped SwiGLU experts whose activations are kept for the backward in
# MXFP8, and MXFP4 experts (32-element blocks along each contraction)
# ---------------------------------------------------------------------------
_HERE = nullcontext()


def _guard(t: Tensor):
    """Makes t's device the current one for the launches of an op, where it is not."""
    return _HERE if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _has_tangent(t: Tensor) -> bool:
    """Whether t carries a derivative of forward mode (a dual tensor, torch.func.jvp's input)."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _check_experts(op: str, x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, counts: Tensor, multiple: int) -> None:
    """The arguments of experts with separate bf16 weights: x [R, D], w1 and w3 [E, H, D],
    w2 [E, D, H], counts [E] integers, all on one device."""
    require_gpu(x, w1, w2, w3, counts)
    _check_bf16(op, x=x, w1=w1, w2=w2, w3=w3)
    xs, ws, cs = x.shape, w1.shape, counts.shape
    if len(xs) != 2 or len(ws) != 3 or len(cs) != 1:
        raise ValueError(f"{op} expects x [R, D], weights [E, .., ..] and counts [E], got {tuple(xs)}, {tuple(ws)}, "
                         f"{tuple(cs)}")
    e, h, d = ws
    if xs[1] != d or w3.shape != ws or w2.shape != (e, d, h) or cs[0] != e:
        raise ValueError(f"{op}: shapes do not agree: x {tuple(xs)}, w1 {tuple(ws)}, w2 {tuple(w2.shape)}, "
                         f"w3 {tuple(w3.shape)}, counts {tuple(cs)}")
    _check_dims(op, e, d, h, multiple)
    _check_counts(op, counts, x, w1, w2, w3)
    if any([_has_tangent(t) for t in (x, w1, w2, w3)]):
        raise RuntimeError(f"{op} has no derivatives in forward mode")


def _check_dims(op: str, e: int, d: int, h: int, multiple: int) -> None:
    if e < 1 or e > MAX_GEMM_EXPERTS:
        raise ValueError(f"{op} takes 1 to {MAX_GEMM_EXPERTS} experts, got {e}")
    if d < multiple or h < multiple or d % multiple or h % multiple:
        raise ValueError(f"{op} takes dims that are multiples of {multiple}, got {d} and {h}")


def _check_counts(op: str, counts: Tensor, *others: Tensor) -> None:
    if counts.is_floating_point() or counts.is_complex() or counts.dtype == torch.bool:
        raise TypeError(f"{op} expects integer counts, got {counts.dtype}")
    here = counts.device
    if any([t.device != here for t in others]):
        raise ValueError(f"{op}: tensors on more than one device")


def _zero_rows_past(counts: Tensor, r: int, e: int, t: Tensor, s: int) -> None:
    # (pairs of bf16 as one word; the dims of the bf16 GEMMs are even)
    call("moe_zero_rows_past_f32", ptr(counts), r, e, ptr(t), t.shape[1] // 2, None, 0, None, 0, None, 0, s)


def _carve(sizes) -> tuple[tuple[int, ...], int]:
    """Offsets of regions of these many bytes in one allocation, each on a 256-byte boundary (the
    kernels' wide loads; whole cache lines), and its size. One kept tensor and one workspace in
    place of 6 to 14 take an eighth to a quarter off a small step's host time (145 -> 125 us of
    grouped_swiglu_ckpt8's forward and backward, 200 -> 147 of grouped_swiglu_mxfp4_train's)."""
    offsets, at = [], 0
    for n in sizes:
        offsets.append(at)
        at += (n + 255) // 256 * 256
    return tuple(offsets), at


@functools.lru_cache(maxsize=256)
def _ckpt8_layout(r: int, d: int, h: int) -> tuple[tuple[int, ...], int]:
    """grouped_swiglu_ckpt8's kept tensor: x [r, d], g and u [r, h] in MXFP8, each with its scales."""
    return _carve(n for c in (d, h, h) for n in (r * c, r * c // MX_BLOCK))


def _at(t: Tensor, offsets) -> list[int]:
    base = t.data_ptr()
    return [base + o for o in offsets]


def _check_kept(op: str, kept: Tensor, size: int, like: Tensor) -> Tensor:
    if kept.dtype is not torch.uint8:
        raise TypeError(f"{op} expects the forward's kept uint8 tensor, got {kept.dtype}")
    if kept.shape != (size,) or kept.device != like.device:
        raise ValueError(f"{op} expects the forward's kept tensor of {size} bytes on {like.device}, got "
                         f"{tuple(kept.shape)} on {kept.device}")
    return _ready(kept)


@torch.library.custom_op("moe_mi355x_mx::grouped_swiglu_ckpt8", mutates_args=())
def grouped_swiglu_ckpt8(
    x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor, for_backward: bool = True
) -> tuple[Tensor, Tensor]:
    """bf16 grouped SwiGLU whose backward works from 8-bit activations. y [R, D] = h w2^T with
    h = bf16(silu(x w1^T) (x w3^T)) of fp32 sums (grouped_swiglu, which follows the reference's,
    rounds four times on the way to h), zero on rows past sum(counts). Then what is kept, as one
    tensor of bytes: x [R, D], g and u [R, H] in MXFP8 (e4m3, one e8m0 scale per 32 along the
    row), each followed by its scales: (D + 2H) 33/32 bytes a row instead of 2D + 6H; empty
    without `for_backward`. The gradients are those at the kept values: the activation's at g and
    u, dw1 and dw3 with x, dw2 with h = silu(g) u; dg, du and that h are taken in fp32 and rounded
    to bf16 once for the products that follow. An infinity or NaN makes its block of 32 kept
    values NaN."""
    op = "grouped_swiglu_ckpt8"
    _check_experts(op, x, w1, w2, w3, num_tokens_per_expert, 64)
    x, w1, w2, w3 = map(_ready, (x, w1, w2, w3))
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h_dim, _ = w1.shape
    offsets, size = _ckpt8_layout(r, d, h_dim)
    kept = x.new_empty(size if for_backward else 0, dtype=torch.uint8)
    x8, xs, g8, gs, up8, us = _at(kept, offsets) if for_backward else (None,) * 6
    h = x.new_empty(r, h_dim)
    y = x.new_empty(r, d)
    with _guard(x):
        s = stream_of(x)
        if for_backward:
            call("moe_keep8_rows", ptr(x), r, d, x8, xs, s)
        call("moe_grouped_gemm_gate_up_keep8", ptr(x), ptr(w1), ptr(w3), ptr(counts), r, e, d, h_dim, g8, gs, up8, us,
             ptr(h), s)
        call("moe_grouped_gemm_down", ptr(h), ptr(w2), ptr(counts), r, e, d, h_dim, ptr(y), s)
        _zero_rows_past(counts, r, e, y, s)
    return y, kept


@grouped_swiglu_ckpt8.register_fake
def _(x, w1, w2, w3, num_tokens_per_expert, for_backward=True):
    size = _ckpt8_layout.__wrapped__(x.shape[0], x.shape[1], w1.shape[1])[1] if for_backward else 0
    return x.new_empty(x.shape), x.new_empty(size, dtype=torch.uint8)


def _narrow_backward(dy: Tensor, e: int, h_dim: int, w1: int, w2: int, w3: int, counts: Tensor, g8: int, gs: int, up8: int,
                     us: int, dgu: int, rows, h: int | None, hidden_kept: bool, need_dx: bool, need_dw13: bool,
                     need_dw2: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """dx, dw1, dw2, dw3 of experts with bf16 weight values and g, u kept in MXFP8, all given by
    address: dgu [R, 2H] is workspace, h [R, H] the forward's (hidden_kept) or where silu(g) u of
    the kept values goes; rows() gives the forward's x. What is not needed comes back empty."""
    r, d = dy.shape
    s = stream_of(dy)
    if need_dx or need_dw13 or not hidden_kept:
        call("moe_grouped_gemm_bwd_dgu_keep8", ptr(dy), w2, g8, gs, up8, us, ptr(counts), r, e, d, h_dim, dgu,
             None if hidden_kept else h, s)
    dx = dy.new_empty(r, d) if need_dx else dy.new_empty(0)
    if need_dx:
        call("moe_grouped_gemm_bwd_dx_once", dgu, w1, w3, ptr(counts), r, e, d, h_dim, ptr(dx), s)
        _zero_rows_past(counts, r, e, dx, s)
    dw1, dw3 = (dy.new_empty((e, h_dim, d) if need_dw13 else 0) for _ in range(2))
    if need_dw13:
        call("moe_grouped_gemm_bwd_dw13", dgu, rows(), ptr(counts), r, e, d, h_dim, ptr(dw1), ptr(dw3), s)
    dw2 = dy.new_empty((e, d, h_dim) if need_dw2 else 0)
    if need_dw2:
        call("moe_grouped_gemm_bwd_dw2", ptr(dy), h, ptr(counts), r, e, d, h_dim, ptr(dw2), s)
    return dx, dw1, dw2, dw3


def _narrow_backward_fake(dy, e, h_dim, need_dx, need_dw13, need_dw2):
    r, d = dy.shape
    bf = lambda need, *shape: dy.new_empty(shape if need else (0,), dtype=torch.bfloat16)  # noqa: E731
    return bf(need_dx, r, d), bf(need_dw13, e, h_dim, d), bf(need_dw2, e, d, h_dim), bf(need_dw13, e, h_dim, d)


@torch.library.custom_op("moe_mi355x_mx::grouped_swiglu_ckpt8_backward", mutates_args=())
def grouped_swiglu_ckpt8_backward(
    dy: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor, kept: Tensor, need_dx: bool = True,
    need_dw13: bool = True, need_dw2: bool = True,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(dx, dw1, dw2, dw3) of grouped_swiglu_ckpt8 from what it kept; dx is zero on rows past
    sum(counts), weights of experts without rows get zeros. What is not needed is empty."""
    op = "grouped_swiglu_ckpt8_backward"
    _check_experts(op, dy, w1, w2, w3, num_tokens_per_expert, 64)
    r, (e, h_dim, d) = dy.shape[0], w1.shape
    offsets, size = _ckpt8_layout(r, d, h_dim)
    kept = _check_kept(op, kept, size, dy)
    dy, w1, w2, w3 = map(_ready, (dy, w1, w2, w3))
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    x8, xs, g8, gs, up8, us = _at(kept, offsets)
    parts, size = _carve((4 * r * h_dim, 2 * r * h_dim if need_dw2 else 0, 2 * r * d if need_dw13 else 0))
    ws = dy.new_empty(size, dtype=torch.uint8)
    dgu, h, x = _at(ws, parts)

    def rows() -> int:
        call("moe_restore8_rows", x8, xs, r, d, x, stream_of(dy))
        return x

    with _guard(dy):
        return _narrow_backward(dy, e, h_dim, ptr(w1), ptr(w2), ptr(w3), counts, g8, gs, up8, us, dgu, rows,
                                h if need_dw2 else None, False, need_dx, need_dw13, need_dw2)


@grouped_swiglu_ckpt8_backward.register_fake
def _(dy, w1, w2, w3, num_tokens_per_expert, kept, need_dx=True, need_dw13=True, need_dw2=True):
    return _narrow_backward_fake(dy, w1.shape[0], w1.shape[1], need_dx, need_dw13, need_dw2)


def _ckpt8_setup(ctx, inputs, output):
    _x, w1, w2, w3, counts, ctx.for_backward = inputs
    ctx.save_for_backward(w1, w2, w3, counts, output[1])
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _needed(need, grads) -> tuple:
    """(dx, dw1, dw2, dw3) with None for inputs that take no gradient."""
    return tuple(g if n else None for n, g in zip(need[:4], grads))


def _ckpt8_bwd(ctx, dy, *_unused):
    if dy is None:
        return (None,) * 6
    if not ctx.for_backward:
        raise RuntimeError("grouped_swiglu_ckpt8 ran with for_backward=False: nothing was kept for a backward")
    need = ctx.needs_input_grad
    return *_needed(need, grouped_swiglu_ckpt8_backward(dy, *ctx.saved_tensors, need[0], need[1] or need[3], need[2])), None, None


grouped_swiglu_ckpt8.register_autograd(_ckpt8_bwd, setup_context=_ckpt8_setup)


# The ops without a gradient are defined on the dispatcher directly: a generation step calls
# them every few microseconds, and without torch.library.custom_op's layers a call takes the host
# 10 us instead of 13 (mxfp4_quantize) and 23 instead of 25 (grouped_swiglu_mxfp4).
_MX = torch.library.Library("moe_mi355x_mx", "FRAGMENT")


# The kernels of the experts' inference, which drop gradients: behind the ops of the same names in
# moe_mi355x_mx and this module, which refuse them.
_MX_BARE = torch.library.Library("moe_mi355x_mx_bare", "FRAGMENT")


def _mx_op(schema: str, lib: torch.library.Library = _MX):
    """Defines the op of this schema in lib with the decorated function as its GPU kernel (and on the
    CPU, where the kernel's own check refuses)."""
    def register(fn):
        name = schema.split("(")[0]
        lib.define(schema)
        lib.impl(name, fn, "CUDA")
        lib.impl(name, fn, "CPU")
        return getattr(getattr(torch.ops, lib.ns), name).default
    return register


def _inference_op(bare, lib: torch.library.Library = _MX):
    """Defines lib's op of the bare one's name and schema as the decorated function, above
    autograd and torch.func's transforms, where it sees what it has to refuse."""
    def register(fn):
        lib.define(str(bare._schema).split("::")[1])
        lib.impl(fn.__name__, fn, "CompositeImplicitAutograd")
        return fn
    return register


def _ready(t: Tensor) -> Tensor:
    """t contiguous and aligned for the kernels."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else _aligned(t.contiguous())


def _mx_dtype(op: str, dtype: torch.dtype) -> int:
    if dtype not in DTYPE_CODES:
        raise TypeError(f"{op} supports bfloat16 and float32, got {dtype}")
    return DTYPE_CODES[dtype]


def _check_mx_matrix(op: str, cols: int) -> None:
    if cols < MX_BLOCK or cols % MX_BLOCK:
        raise ValueError(f"{op} takes rows of whole blocks of {MX_BLOCK} elements, got {cols}")


def _check_packed(op: str, name: str, q: Tensor, scale: Tensor, shape: tuple | None = None) -> None:
    """An MXFP4 matrix: q [.., K / 2] and scale [.., K / 32] bytes on one device, of the values'
    `shape` where one is given."""
    if q.dtype != torch.uint8 or scale.dtype != torch.uint8:
        raise TypeError(f"{op} expects uint8 {name} and scales, got {q.dtype} and {scale.dtype}")
    qs, ss = q.shape, scale.shape
    if not qs or len(ss) != len(qs) or ss[:-1] != qs[:-1] or q.device != scale.device:
        raise ValueError(f"{op}: {name} {tuple(qs)} on {q.device} and its scales {tuple(ss)} on "
                         f"{scale.device} do not belong together")
    _check_mx_matrix(op, 2 * qs[-1])
    if ss[-1] * 16 != qs[-1]:
        raise ValueError(f"{op}: {name} of {2 * qs[-1]} columns takes {qs[-1] // 16} scales a row, got {ss[-1]}")
    if shape is not None and (*qs[:-1], 2 * qs[-1]) != shape:
        raise ValueError(f"{op} expects {name} of {list(shape)} values, got {[*qs[:-1], 2 * qs[-1]]}")


@_mx_op("mxfp4_quantize(Tensor x) -> (Tensor, Tensor)")
def _mxfp4_quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    require_gpu(x)
    code = _mx_dtype("mxfp4_quantize", x.dtype)
    if x.dim() < 1:
        raise ValueError("mxfp4_quantize expects rows, got a scalar")
    *lead, cols = x.shape
    _check_mx_matrix("mxfp4_quantize", cols)
    x = _ready(x)
    q = x.new_empty(*lead, cols // 2, dtype=torch.uint8)
    scale = x.new_empty(*lead, cols // MX_BLOCK, dtype=torch.uint8)
    with _guard(x):
        call("moe_mxfp4_quant_rows", ptr(x), x.numel() // cols, cols, cols, code, ptr(q), ptr(scale), stream_of(x))
    return q, scale


@torch.library.register_fake("moe_mi355x_mx::mxfp4_quantize", lib=_MX)
def _(x):
    u8 = lambda n: x.new_empty(*x.shape[:-1], n, dtype=torch.uint8)  # noqa: E731
    return u8(x.shape[-1] // 2), u8(x.shape[-1] // MX_BLOCK)


def mxfp4_quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    """x [.., K] (bf16 or fp32, K a multiple of 32) in MXFP4: (q [.., K / 2] uint8, two e2m1
    codes a byte, the first in the low half; scale [.., K / 32] uint8, e8m0). A block's scale is
    the least power of two 2^k, k in [-127, 127], with max |x| <= 6 * 2^k; elements are rounded
    to nearest, ties to the even code. A block with an infinity or a NaN gets the NaN scale 255."""
    return _mxfp4_quantize(x.detach())


@_mx_op("mxfp4_dequantize(Tensor q, Tensor scale, ScalarType dtype) -> Tensor")
def _mxfp4_dequantize(q: Tensor, scale: Tensor, dtype: torch.dtype) -> Tensor:
    require_gpu(q, scale)
    code = _mx_dtype("mxfp4_dequantize", dtype)
    _check_packed("mxfp4_dequantize", "q", q, scale)
    *lead, half = q.shape
    q, scale = _ready(q), scale.contiguous()
    x = q.new_empty(*lead, 2 * half, dtype=dtype)
    with _guard(q):
        call("moe_mxfp4_dequant_rows", ptr(q), ptr(scale), q.numel() // half, 2 * half, 2 * half, code, ptr(x), stream_of(q))
    return x


@torch.library.register_fake("moe_mi355x_mx::mxfp4_dequantize", lib=_MX)
def _(q, scale, dtype):
    return q.new_empty(*q.shape[:-1], 2 * q.shape[-1], dtype=dtype)


def mxfp4_dequantize(q: Tensor, scale: Tensor, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The values [.., K] of an MXFP4 matrix (q [.., K / 2], scale [.., K / 32] uint8) in bf16 or
    fp32, which hold each of them exactly within their range (past it: infinities)."""
    return _mxfp4_dequantize(q, scale, dtype)


@functools.lru_cache(maxsize=256)
def _mxfp4_workspace_bytes(r: int, e: int, d: int, h_dim: int) -> int:
    return max(int(lib().moe_mxfp4_workspace_bytes(r, e, d, h_dim)), 16)


def _check_mxfp4_rows(op: str, x: Tensor, qw1: Tensor, counts: Tensor, glu: int = 1) -> tuple[int, int, int, int]:
    _check_bf16(op, x=x)
    xs, ws, cs = x.shape, qw1.shape, counts.shape
    if len(xs) != 2 or len(ws) != 3 or len(cs) != 1 or cs[0] != ws[0] or ws[1] % glu:
        raise ValueError(f"{op} expects x [R, D], packed weights [E, .., ..] and counts [E], got {tuple(xs)}, "
                         f"{tuple(ws)}, {tuple(cs)}")
    r, d = xs
    e, h_dim = ws[0], ws[1] // glu
    _check_dims(op, e, d, h_dim, MX_BLOCK)
    return r, d, e, h_dim


def _no_gradients(op: str, *tensors: Tensor | None, instead: str = "grouped_swiglu_mxfp4_train trains on bf16 weights") -> None:
    grad = torch.is_grad_enabled()
    if any([t is not None and ((grad and t.requires_grad) or _has_tangent(t)) for t in tensors]):
        raise RuntimeError(f"{op} is for inference and has no gradients: call it under torch.no_grad() or on detached "
                           f"tensors ({instead})")


@_mx_op("grouped_swiglu_mxfp4(Tensor x, Tensor qw1, Tensor sw1, Tensor qw2, Tensor sw2, Tensor qw3, Tensor sw3, "
        "Tensor num_tokens_per_expert) -> Tensor", _MX_BARE)
def _grouped_swiglu_mxfp4(x, qw1, sw1, qw2, sw2, qw3, sw3, num_tokens_per_expert):
    op = "grouped_swiglu_mxfp4"
    counts = num_tokens_per_expert
    require_gpu(x, qw1, sw1, qw2, sw2, qw3, sw3, counts)
    r, d, e, h_dim = _check_mxfp4_rows(op, x, qw1, counts)
    _check_packed(op, "w1", qw1, sw1, (e, h_dim, d))
    _check_packed(op, "w2", qw2, sw2, (e, d, h_dim))
    _check_packed(op, "w3", qw3, sw3, (e, h_dim, d))
    _check_counts(op, counts, x, qw1, qw2, qw3)
    x, qw1, sw1, qw2, sw2, qw3, sw3 = map(_ready, (x, qw1, sw1, qw2, sw2, qw3, sw3))
    counts = counts.to(torch.int64).contiguous()
    ws_bytes = _mxfp4_workspace_bytes(r, e, d, h_dim)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    y = x.new_empty(r, d)
    with _guard(x):
        call("moe_mxfp4_swiglu_fwd", ptr(x), ptr(qw1), ptr(sw1), ptr(qw2), ptr(sw2), ptr(qw3), ptr(sw3), ptr(counts), r, e,
             d, h_dim, ptr(ws), ws_bytes, ptr(y), stream_of(x))
    return y


@torch.library.register_fake("moe_mi355x_mx_bare::grouped_swiglu_mxfp4", lib=_MX_BARE)
def _(x, qw1, sw1, qw2, sw2, qw3, sw3, num_tokens_per_expert):
    return x.new_empty(x.shape)


@_inference_op(_grouped_swiglu_mxfp4)
def grouped_swiglu_mxfp4(
    x: Tensor, qw1: Tensor, sw1: Tensor, qw2: Tensor, sw2: Tensor, qw3: Tensor, sw3: Tensor,
    num_tokens_per_expert: Tensor,
) -> Tensor:
    """The SwiGLU experts on weights packed in MXFP4 (mxfp4_quantize of w1, w3 [E, H, D] and
    w2 [E, D, H]): x [R, D] bf16 in expert order is quantized on the way, h = silu(x w1^T)
    (x w3^T) is taken in fp32 and quantized, y = h w2^T [R, D] is rounded to bf16 once. Rows past
    sum(counts) are zero. For inference: no gradients. D and H are multiples of 32."""
    _no_gradients("grouped_swiglu_mxfp4", x)
    return _grouped_swiglu_mxfp4(x, qw1, sw1, qw2, sw2, qw3, sw3, num_tokens_per_expert)


@_mx_op("grouped_swiglu_oss_mxfp4(Tensor x, Tensor qmlp1, Tensor smlp1, Tensor mlp1_bias, Tensor qmlp2, Tensor smlp2, "
        "Tensor mlp2_bias, Tensor num_tokens_per_expert, float swiglu_limit) -> Tensor", _MX_BARE)
def _grouped_swiglu_oss_mxfp4(x, qmlp1, smlp1, mlp1_bias, qmlp2, smlp2, mlp2_bias, num_tokens_per_expert, swiglu_limit):
    op = "grouped_swiglu_oss_mxfp4"
    counts = num_tokens_per_expert
    require_gpu(x, qmlp1, smlp1, mlp1_bias, qmlp2, smlp2, mlp2_bias, counts)
    r, d, e, h_dim = _check_mxfp4_rows(op, x, qmlp1, counts, 2)
    _check_packed(op, "mlp1", qmlp1, smlp1, (e, 2 * h_dim, d))
    _check_packed(op, "mlp2", qmlp2, smlp2, (e, d, h_dim))
    if tuple(mlp1_bias.shape) != (e, 2 * h_dim) or tuple(mlp2_bias.shape) != (e, d):
        raise ValueError(f"{op} expects biases [{e}, {2 * h_dim}] and [{e}, {d}], got {tuple(mlp1_bias.shape)} and "
                         f"{tuple(mlp2_bias.shape)}")
    if not swiglu_limit >= 0:
        raise ValueError(f"{op} expects a clamp limit of at least 0, got {swiglu_limit}")
    _check_counts(op, counts, x, qmlp1, mlp1_bias, qmlp2, mlp2_bias)
    x, qmlp1, smlp1, qmlp2, smlp2 = map(_ready, (x, qmlp1, smlp1, qmlp2, smlp2))
    b1, b2 = _ready(mlp1_bias.to(torch.bfloat16)), _ready(mlp2_bias.to(torch.bfloat16))
    counts = counts.to(torch.int64).contiguous()
    ws_bytes = _mxfp4_workspace_bytes(r, e, d, h_dim)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    y = x.new_empty(r, d)
    with _guard(x):
        call("moe_mxfp4_oss_fwd", ptr(x), ptr(qmlp1), ptr(smlp1), ptr(b1), ptr(qmlp2), ptr(smlp2), ptr(b2), ptr(counts), r,
             e, d, h_dim, float(swiglu_limit), ptr(ws), ws_bytes, ptr(y), stream_of(x))
    return y


@torch.library.register_fake("moe_mi355x_mx_bare::grouped_swiglu_oss_mxfp4", lib=_MX_BARE)
def _(x, qmlp1, smlp1, mlp1_bias, qmlp2, smlp2, mlp2_bias, num_tokens_per_expert, swiglu_limit):
    return x.new_empty(x.shape)


@_inference_op(_grouped_swiglu_oss_mxfp4)
def grouped_swiglu_oss_mxfp4(
    x: Tensor, qmlp1: Tensor, smlp1: Tensor, mlp1_bias: Tensor, qmlp2: Tensor, smlp2: Tensor, mlp2_bias: Tensor,
    num_tokens_per_expert: Tensor, swiglu_limit: float,
) -> Tensor:
    """grouped_swiglu_mxfp4 for gpt-oss's experts (gpt_oss/moe.py:43-122): mlp1 [E, 2H, D] (glu row
    2j, linear row 2j + 1) and mlp2 [E, D, H] packed in MXFP4, biases [E, 2H] and [E, D] taken in
    bf16; biases, clamps and activation in fp32 between the products."""
    _no_gradients("grouped_swiglu_oss_mxfp4", x, mlp1_bias, mlp2_bias)
    return _grouped_swiglu_oss_mxfp4(x, qmlp1, smlp1, mlp1_bias, qmlp2, smlp2, mlp2_bias, num_tokens_per_expert,
                                     swiglu_limit)


def _mxfp4_padded(cols: int) -> int:  # moe_mxfp4_padded_cols
    return (cols + 255) // 256 * 256


@functools.lru_cache(maxsize=256)
def _mxfp4_train_layout(r: int, e: int, d: int, h: int) -> tuple[tuple[int, ...], int]:
    """grouped_swiglu_mxfp4_train's kept tensor: w1, w2, w3, x and h in MXFP4 (the rows of x and h
    padded to 256 columns, zeros behind), g and u in MXFP8, each with its scales."""
    w = e * d * h
    four = [n for c in (w, w, w, r * _mxfp4_padded(d), r * _mxfp4_padded(h)) for n in (c // 2, c // MX_BLOCK)]
    return _carve(four + [n for c in (r * h, r * h) for n in (c, c // MX_BLOCK)])


@torch.library.custom_op("moe_mi355x_mx::grouped_swiglu_mxfp4_train", mutates_args=())
def grouped_swiglu_mxfp4_train(
    x: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor
) -> tuple[Tensor, Tensor]:
    """The SwiGLU experts in MXFP4 from bf16 weights, with gradients: y [R, D] is
    grouped_swiglu_mxfp4's on the packed weights. The backward passes the quantizations
    straight through: it takes the products' gradients at their quantized operands (in bf16,
    which holds them exactly) and the activation's at g and u kept in MXFP8, in fp32, with dg and du
    rounded to bf16 once for the products that follow. Returns y, then what is kept, as one tensor of bytes: w1, w2, w3, x and h in MXFP4 and g, u in MXFP8, each
    with its scales. D and H are multiples of 64."""
    op = "grouped_swiglu_mxfp4_train"
    _check_experts(op, x, w1, w2, w3, num_tokens_per_expert, 64)
    x, w1, w2, w3 = map(_ready, (x, w1, w2, w3))
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    r, d = x.shape
    e, h_dim, _ = w1.shape
    offsets, size = _mxfp4_train_layout(r, e, d, h_dim)
    kept = x.new_empty(size, dtype=torch.uint8)
    qw1, sw1, qw2, sw2, qw3, sw3, qx, sx, qh, sh, g8, gs, up8, us = _at(kept, offsets)
    y = x.new_empty(r, d)
    with _guard(x):
        s = stream_of(x)
        call("moe_mxfp4_quant_rows", ptr(x), r, d, _mxfp4_padded(d), 0, qx, sx, s)
        for w, q, sc, rows, cols in ((w1, qw1, sw1, e * h_dim, d), (w2, qw2, sw2, e * d, h_dim), (w3, qw3, sw3, e * h_dim, d)):
            call("moe_mxfp4_quant_rows", ptr(w), rows, cols, cols, 0, q, sc, s)
        call("moe_mxfp4_gemm_gate_up_keep", qx, sx, qw1, sw1, qw3, sw3, ptr(counts), r, e, d, h_dim, qh, sh, g8, gs, up8, us,
             s)
        call("moe_mxfp4_gemm_down", qh, sh, qw2, sw2, ptr(counts), r, e, d, h_dim, ptr(y), s)
    return y, kept


@grouped_swiglu_mxfp4_train.register_fake
def _(x, w1, w2, w3, num_tokens_per_expert):
    e, h_dim, d = w1.shape
    size = _mxfp4_train_layout.__wrapped__(x.shape[0], e, d, h_dim)[1]
    return x.new_empty(x.shape), x.new_empty(size, dtype=torch.uint8)


@torch.library.custom_op("moe_mi355x_mx::grouped_swiglu_mxfp4_train_backward", mutates_args=())
def grouped_swiglu_mxfp4_train_backward(
    dy: Tensor, num_tokens_per_expert: Tensor, kept: Tensor, hidden_dim: int, need_dx: bool = True, need_dw13: bool = True,
    need_dw2: bool = True,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(dx, dw1, dw2, dw3) of grouped_swiglu_mxfp4_train from what it kept; dx is zero on rows
    past sum(counts), weights of experts without rows get zeros. What is not needed is empty."""
    op = "grouped_swiglu_mxfp4_train_backward"
    counts, h_dim = num_tokens_per_expert, hidden_dim
    require_gpu(dy, counts)
    _check_bf16(op, dy=dy)
    if dy.dim() != 2 or counts.dim() != 1:
        raise ValueError(f"{op} expects dy [R, D] and counts [E], got {tuple(dy.shape)}, {tuple(counts.shape)}")
    (r, d), e = dy.shape, counts.shape[0]
    _check_dims(op, e, d, h_dim, 64)
    _check_counts(op, counts, dy)
    offsets, size = _mxfp4_train_layout(r, e, d, h_dim)
    kept = _check_kept(op, kept, size, dy)
    dy, counts = _ready(dy), counts.to(torch.int64).contiguous()
    qw1, sw1, qw2, sw2, qw3, sw3, qx, sx, qh, sh, g8, gs, up8, us = _at(kept, offsets)
    need_dgu, n_w = need_dx or need_dw13, 2 * e * d * h_dim
    parts, size = _carve((n_w if need_dx else 0, n_w if need_dgu else 0, n_w if need_dx else 0,
                          4 * r * h_dim if need_dgu else 0, 2 * r * h_dim if need_dw2 else 0, 2 * r * d if need_dw13 else 0))
    ws = dy.new_empty(size, dtype=torch.uint8)
    w1, w2, w3, dgu, h, x = _at(ws, parts)

    def values(q: int, scale: int, rows: int, cols: int, q_cols: int, out: int) -> int:
        call("moe_mxfp4_dequant_rows", q, scale, rows, cols, q_cols, 0, out, stream_of(dy))
        return out

    with _guard(dy):
        if need_dgu:
            values(qw2, sw2, e * d, h_dim, h_dim, w2)
        if need_dx:
            values(qw1, sw1, e * h_dim, d, d, w1)
            values(qw3, sw3, e * h_dim, d, d, w3)
        if need_dw2:
            values(qh, sh, r, h_dim, _mxfp4_padded(h_dim), h)
        return _narrow_backward(dy, e, h_dim, w1, w2, w3, counts, g8, gs, up8, us, dgu,
                                lambda: values(qx, sx, r, d, _mxfp4_padded(d), x), h, True, need_dx, need_dw13, need_dw2)


@grouped_swiglu_mxfp4_train_backward.register_fake
def _(dy, num_tokens_per_expert, kept, hidden_dim, need_dx=True, need_dw13=True, need_dw2=True):
    return _narrow_backward_fake(dy, num_tokens_per_expert.shape[0], hidden_dim, need_dx, need_dw13, need_dw2)


def _mxfp4_train_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[4], output[1])
    ctx.mark_non_differentiable(output[1])
    ctx.hidden_dim = inputs[1].shape[1]
    ctx.set_materialize_grads(False)


def _mxfp4_train_bwd(ctx, dy, *_unused):
    if dy is None:
        return None, None, None, None, None
    need = ctx.needs_input_grad
    return *_needed(need, grouped_swiglu_mxfp4_train_backward(dy, *ctx.saved_tensors, ctx.hidden_dim, need[0],
                                                              need[1] or need[3], need[2])), None


grouped_swiglu_mxfp4_train.register_autograd(_mxfp4_train_bwd, setup_context=_mxfp4_train_setup)


# ---------------------------------------------------------------------------
# 8-bit integers with a scale per row (token or output channel), for inference
# ---------------------------------------------------------------------------
_I8 = torch.library.Library("moe_mi355x_int8", "FRAGMENT")
_I8_BARE = torch.library.Library("moe_mi355x_int8_bare", "FRAGMENT")  # (as _MX_BARE)
INT8_MULTIPLE = 16  # of the products' contractions: weight rows are read in 16-byte pieces
INT8_MAX_K = 131072  # past it a sum of code products can leave 32 bits
INT8_MAX_COLUMNS = 2 ** 30  # of rows by themselves
INT8_MAX_N = 2 ** 22  # output channels

# A generation step's calls take the host as long as the GPU, so what is right is checked in few
# steps, and a message is put together where something is not.


def _int8_device(op: str, x: Tensor, *others: Tensor | None) -> int:
    """The GPU that all of them are on."""
    here = x.get_device()
    ok = here >= 0
    for t in others:
        if t is not None and t.get_device() != here:
            ok = False
    if not ok:
        require_gpu(x, *others)
        raise ValueError(f"{op}: tensors on more than one device")
    return here


def _int8_launch(here: int, name: str, x: Tensor, *args) -> None:
    """An entry point on x's device and torch's stream there."""
    if here == torch._C._cuda_getDevice():
        call(name, *args, stream_of(x))
    else:
        with torch.cuda.device(here):
            call(name, *args, stream_of(x))


def _check_int8(op: str, name: str, q: Tensor, scale: Tensor, shape: tuple) -> None:
    """A matrix in codes: q of `shape` int8 and scale of shape[:-1] fp32."""
    if q.dtype is torch.int8 and scale.dtype is torch.float32 and q.shape == shape and scale.shape == shape[:-1]:
        return
    if q.dtype is not torch.int8 or scale.dtype is not torch.float32:
        raise TypeError(f"{op} expects int8 {name} and float32 scales, got {q.dtype} and {scale.dtype}")
    raise ValueError(f"{op} expects {name} of {list(shape)} with scales of {list(shape[:-1])}, got {list(q.shape)} and "
                     f"{list(scale.shape)}")


def _check_int8_bias(op: str, bias: Tensor, shape: tuple) -> int:
    """The bias's dtype code."""
    if bias.dtype not in DTYPE_CODES:
        raise TypeError(f"{op} takes biases in bfloat16 and float32, got {bias.dtype}")
    if bias.shape != shape:
        raise ValueError(f"{op} expects a bias of {list(shape)}, got {list(bias.shape)}")
    return DTYPE_CODES[bias.dtype]


def _check_int8_dims(op: str, e: int, *contractions: int) -> None:
    if e < 1 or e > MAX_GEMM_EXPERTS:
        raise ValueError(f"{op} takes 1 to {MAX_GEMM_EXPERTS} experts, got {e}")
    for k in contractions:
        if k < INT8_MULTIPLE or k % INT8_MULTIPLE or k > INT8_MAX_K:
            raise ValueError(f"{op} takes contractions that are multiples of {INT8_MULTIPLE} up to {INT8_MAX_K}, got {k}")


def _int8_code(op: str, dtype: torch.dtype) -> int:
    code = DTYPE_CODES.get(dtype)
    if code is None:
        raise TypeError(f"{op} supports bfloat16 and float32, got {dtype}")
    return code


def _check_int8_columns(op: str, rows: Tensor) -> None:
    if not rows.dim() or not 1 <= rows.shape[-1] <= INT8_MAX_COLUMNS:
        raise ValueError(f"{op} expects rows of 1 to {INT8_MAX_COLUMNS} columns, got {tuple(rows.shape)}")


def _no_int8_gradients(op: str, *tensors: Tensor | None) -> None:
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and (t.requires_grad or forward_ad._current_level >= 0):
                _no_gradients(op, t, instead="codes are not differentiable: train on the bf16 weights")


@_mx_op("int8_quantize(Tensor x) -> (Tensor, Tensor)", _I8_BARE)
def _int8_quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    here = _int8_device("int8_quantize", x)
    code = _int8_code("int8_quantize", x.dtype)
    _check_int8_columns("int8_quantize", x)
    shape = x.shape
    ld = cols = shape[-1]
    if not x.is_contiguous():
        if len(shape) == 2 and x.stride(1) == 1 and x.stride(0) >= cols:
            ld = x.stride(0)  # a slice of wider rows is read where it is
        else:
            x = x.contiguous()
    q = torch.empty_like(x, dtype=torch.int8) if ld == cols else x.new_empty(shape, dtype=torch.int8)
    scale = x.new_empty(shape[:-1], dtype=torch.float32)
    _int8_launch(here, "moe_int8_quant_rows", x, x.data_ptr(), ld, scale.numel(), cols, code, q.data_ptr(), scale.data_ptr())
    return q, scale


@torch.library.register_fake("moe_mi355x_int8_bare::int8_quantize", lib=_I8_BARE)
def _(x):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


@_inference_op(_int8_quantize, _I8)
def int8_quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    """x [.., K] (bf16 or fp32) in 8-bit integers with a scale for each row: (q [.., K] int8,
    scale [..] fp32). With a = max(max |x|, 127 * 2^-126) of a row and the fp32 quotients
    r = 127 / a, scale = a / 127, its codes are x r rounded once to the nearest integer, ties to
    even (|q| <= 127), and stand for q scale. A row with an infinity or a NaN has the scale NaN
    and zero codes. Rows of weights [.., N, K] are output channels, rows of activations tokens. For
    inference: no gradients."""
    _no_int8_gradients("int8_quantize", x)
    return _int8_quantize(x)


@_mx_op("int8_dequantize(Tensor q, Tensor scale, ScalarType dtype) -> Tensor", _I8_BARE)
def _int8_dequantize(q: Tensor, scale: Tensor, dtype: torch.dtype) -> Tensor:
    here = _int8_device("int8_dequantize", q, scale)
    code = _int8_code("int8_dequantize", dtype)
    _check_int8_columns("int8_dequantize", q)
    _check_int8("int8_dequantize", "q", q, scale, q.shape)
    q, scale = q.contiguous(), scale.contiguous()
    x = torch.empty_like(q, dtype=dtype)
    _int8_launch(here, "moe_int8_dequant_rows", q, q.data_ptr(), scale.data_ptr(), scale.numel(), q.shape[-1], code, x.data_ptr())
    return x


@torch.library.register_fake("moe_mi355x_int8_bare::int8_dequantize", lib=_I8_BARE)
def _(q, scale, dtype):
    return q.new_empty(q.shape, dtype=dtype)


@_inference_op(_int8_dequantize, _I8)
def int8_dequantize(q: Tensor, scale: Tensor, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The values q scale [.., K] of a matrix in codes (int8_quantize), taken in fp32, in bf16 or
    fp32. For inference: no gradients."""
    _no_int8_gradients("int8_dequantize", scale)
    return _int8_dequantize(q, scale, dtype)


@functools.lru_cache(maxsize=256)
def _int8_linear_workspace_bytes(r: int, e: int, k: int, n: int) -> int:
    return max(int(lib().moe_int8_linear_workspace_bytes(r, e, k, n)), 0)  # (what does not fit, the call refuses)


@functools.lru_cache(maxsize=256)
def _int8_layer_workspace_bytes(r: int, e: int, d: int, h: int) -> int:
    return int(lib().moe_int8_layer_workspace_bytes(r, e, d, h))


def _int8_product(op: str, here: int, x: Tensor, qw: Tensor, sw: Tensor, counts: Tensor | None, bias: Tensor | None,
                  rows: int, e: int, n: int, k: int) -> Tensor:
    """x [.., K] of `rows` rows by qw [(E,) N, K]."""
    code = _int8_code(op, x.dtype)
    _check_int8(op, "qw", qw, sw, qw.shape)
    _check_int8_dims(op, e, k)
    if not 1 <= n <= INT8_MAX_N:
        raise ValueError(f"{op} expects 1 to {INT8_MAX_N} output channels, got {tuple(qw.shape)}")
    bias_code = 0
    if bias is not None:
        bias_code = _check_int8_bias(op, bias, qw.shape[:-1])
        bias = bias.contiguous()
    x, qw, sw = _ready(x), _ready(qw), sw.contiguous()
    ws_bytes = _int8_linear_workspace_bytes(rows, e, k, n)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    y = x.new_empty((*x.shape[:-1], n))
    _int8_launch(here, "moe_int8_linear", x, x.data_ptr(), code, qw.data_ptr(), sw.data_ptr(), ptr(bias), bias_code, ptr(counts),
                 rows, e, k, n, ptr(ws), ws_bytes, y.data_ptr())
    return y


def _rows_of(xs: torch.Size) -> int:
    return xs[0] if len(xs) == 2 else xs[:-1].numel()


@_mx_op("linear_int8(Tensor x, Tensor qw, Tensor sw, Tensor? bias=None) -> Tensor", _I8_BARE)
def _linear_int8(x, qw, sw, bias=None):
    op = "linear_int8"
    here = _int8_device(op, x, qw, sw, bias)
    xs, ws = x.shape, qw.shape
    if len(ws) != 2 or not xs or xs[-1] != ws[1]:
        raise ValueError(f"{op} expects x [.., K] and qw [N, K], got {tuple(xs)} and {tuple(ws)}")
    return _int8_product(op, here, x, qw, sw, None, bias, _rows_of(xs), 1, *ws)


@torch.library.register_fake("moe_mi355x_int8_bare::linear_int8", lib=_I8_BARE)
def _(x, qw, sw, bias=None):
    return x.new_empty(*x.shape[:-1], qw.shape[0])


@_inference_op(_linear_int8, _I8)
def linear_int8(x: Tensor, qw: Tensor, sw: Tensor, bias: Tensor | None = None) -> Tensor:
    """x w^T + bias in x's dtype (bf16 or fp32), for x [.., K] and a weight in codes, qw [N, K]
    int8 with sw [N] (int8_quantize). x's rows are quantized on the way; the sums of code products
    are exact, their scales and the bias (bf16 or fp32) are applied in fp32 and the result is
    rounded once. For inference: no gradients. K is a multiple of 16."""
    _no_int8_gradients("linear_int8", x, sw, bias)
    return _linear_int8(x, qw, sw, bias)


def _int8_counts(op: str, x: Tensor, qw: Tensor, counts: Tensor) -> Tensor:
    """The counts of grouped rows as the kernels read them."""
    xs, ws, cs = x.shape, qw.shape, counts.shape
    if len(xs) != 2 or len(ws) != 3 or len(cs) != 1 or cs[0] != ws[0] or xs[1] != ws[2]:
        raise ValueError(f"{op} expects x [R, K], weights [E, .., K] and counts [E], got {tuple(xs)}, {tuple(ws)}, {tuple(cs)}")
    if counts.dtype is not torch.int64:
        _check_counts(op, counts)
        counts = counts.to(torch.int64)
    return counts.contiguous()


@_mx_op("grouped_linear_int8(Tensor x, Tensor qw, Tensor sw, Tensor num_tokens_per_expert, Tensor? bias=None) -> Tensor",
        _I8_BARE)
def _grouped_linear_int8(x, qw, sw, num_tokens_per_expert, bias=None):
    op = "grouped_linear_int8"
    here = _int8_device(op, x, qw, sw, num_tokens_per_expert, bias)
    counts = _int8_counts(op, x, qw, num_tokens_per_expert)
    return _int8_product(op, here, x, qw, sw, counts, bias, x.shape[0], *qw.shape)


@torch.library.register_fake("moe_mi355x_int8_bare::grouped_linear_int8", lib=_I8_BARE)
def _(x, qw, sw, num_tokens_per_expert, bias=None):
    return x.new_empty(x.shape[0], qw.shape[1])


@_inference_op(_grouped_linear_int8, _I8)
def grouped_linear_int8(x: Tensor, qw: Tensor, sw: Tensor, num_tokens_per_expert: Tensor, bias: Tensor | None = None) -> Tensor:
    """linear_int8 with a weight (and bias) per expert: x [R, K] in expert order, qw [E, N, K], sw and
    bias [E, N], counts [E] -> [R, N]. Rows past sum(counts) are zero."""
    _no_int8_gradients("grouped_linear_int8", x, sw, bias)
    return _grouped_linear_int8(x, qw, sw, num_tokens_per_expert, bias)


def _int8_swiglu(op: str, here: int, x, qw1, sw1, qw2, sw2, qw3, sw3, counts, rows) -> Tensor:
    _check_bf16(op, x=x)
    shape = qw1.shape
    e, h, d = shape if len(shape) == 3 else (1, *shape)
    _check_int8(op, "w1", qw1, sw1, shape)
    _check_int8(op, "w2", qw2, sw2, (e, d, h) if len(shape) == 3 else (d, h))
    _check_int8(op, "w3", qw3, sw3, shape)
    _check_int8_dims(op, e, d, h)
    x, qw1, qw2, qw3 = _ready(x), _ready(qw1), _ready(qw2), _ready(qw3)
    sw1, sw2, sw3 = sw1.contiguous(), sw2.contiguous(), sw3.contiguous()
    ws_bytes = _int8_layer_workspace_bytes(rows, e, d, h)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    y = torch.empty_like(x)
    _int8_launch(here, "moe_int8_swiglu", x, x.data_ptr(), qw1.data_ptr(), sw1.data_ptr(), qw2.data_ptr(), sw2.data_ptr(),
                 qw3.data_ptr(), sw3.data_ptr(), ptr(counts), rows, e, d, h, ws.data_ptr(), ws_bytes, y.data_ptr())
    return y


@_mx_op("swiglu_ffn_int8(Tensor x, Tensor qw1, Tensor sw1, Tensor qw2, Tensor sw2, Tensor qw3, Tensor sw3) -> Tensor", _I8_BARE)
def _swiglu_ffn_int8(x, qw1, sw1, qw2, sw2, qw3, sw3):
    op = "swiglu_ffn_int8"
    here = _int8_device(op, x, qw1, sw1, qw2, sw2, qw3, sw3)
    if qw1.dim() != 2 or x.dim() < 1 or x.shape[-1] != qw1.shape[1]:
        raise ValueError(f"{op} expects x [.., D] and weights [H, D] and [D, H], got {tuple(x.shape)} and {tuple(qw1.shape)}")
    return _int8_swiglu(op, here, x, qw1, sw1, qw2, sw2, qw3, sw3, None, _rows_of(x.shape))


@torch.library.register_fake("moe_mi355x_int8_bare::swiglu_ffn_int8", lib=_I8_BARE)
def _(x, qw1, sw1, qw2, sw2, qw3, sw3):
    return x.new_empty(x.shape)


@_inference_op(_swiglu_ffn_int8, _I8)
def swiglu_ffn_int8(x: Tensor, qw1: Tensor, sw1: Tensor, qw2: Tensor, sw2: Tensor, qw3: Tensor, sw3: Tensor) -> Tensor:
    """The SwiGLU feed-forward on weights in codes: x [.., D] bf16, w1 and w3 [H, D], w2 [D, H]
    (int8_quantize). h = silu(x w1^T) (x w3^T) is taken in fp32 and quantized like x, h w2^T is
    rounded to bf16 once. For inference: no gradients. D and H are multiples of 16."""
    _no_int8_gradients("swiglu_ffn_int8", x, sw1, sw2, sw3)
    return _swiglu_ffn_int8(x, qw1, sw1, qw2, sw2, qw3, sw3)


@_mx_op("grouped_swiglu_int8(Tensor x, Tensor qw1, Tensor sw1, Tensor qw2, Tensor sw2, Tensor qw3, Tensor sw3, "
        "Tensor num_tokens_per_expert) -> Tensor", _I8_BARE)
def _grouped_swiglu_int8(x, qw1, sw1, qw2, sw2, qw3, sw3, num_tokens_per_expert):
    op = "grouped_swiglu_int8"
    here = _int8_device(op, x, qw1, sw1, qw2, sw2, qw3, sw3, num_tokens_per_expert)
    counts = _int8_counts(op, x, qw1, num_tokens_per_expert)
    return _int8_swiglu(op, here, x, qw1, sw1, qw2, sw2, qw3, sw3, counts, x.shape[0])


@torch.library.register_fake("moe_mi355x_int8_bare::grouped_swiglu_int8", lib=_I8_BARE)
def _(x, qw1, sw1, qw2, sw2, qw3, sw3, num_tokens_per_expert):
    return x.new_empty(x.shape)


@_inference_op(_grouped_swiglu_int8, _I8)
def grouped_swiglu_int8(
    x: Tensor, qw1: Tensor, sw1: Tensor, qw2: Tensor, sw2: Tensor, qw3: Tensor, sw3: Tensor,
    num_tokens_per_expert: Tensor,
) -> Tensor:
    """swiglu_ffn_int8 with weights per expert, w1 and w3 [E, H, D], w2 [E, D, H]: x [R, D] bf16 in
    expert order, counts [E]. Rows past sum(counts) are zero."""
    _no_int8_gradients("grouped_swiglu_int8", x, sw1, sw2, sw3)
    return _grouped_swiglu_int8(x, qw1, sw1, qw2, sw2, qw3, sw3, num_tokens_per_expert)


@_mx_op("grouped_swiglu_oss_int8(Tensor x, Tensor qmlp1, Tensor smlp1, Tensor mlp1_bias, Tensor qmlp2, Tensor smlp2, "
        "Tensor mlp2_bias, Tensor num_tokens_per_expert, float swiglu_limit) -> Tensor", _I8_BARE)
def _grouped_swiglu_oss_int8(x, qmlp1, smlp1, mlp1_bias, qmlp2, smlp2, mlp2_bias, num_tokens_per_expert, swiglu_limit):
    op = "grouped_swiglu_oss_int8"
    here = _int8_device(op, x, qmlp1, smlp1, mlp1_bias, qmlp2, smlp2, mlp2_bias, num_tokens_per_expert)
    _check_bf16(op, x=x)
    counts = _int8_counts(op, x, qmlp1, num_tokens_per_expert)
    (r, d), (e, h2, _) = x.shape, qmlp1.shape
    h = h2 // 2
    _check_int8(op, "mlp1", qmlp1, smlp1, (e, 2 * h, d))
    _check_int8(op, "mlp2", qmlp2, smlp2, (e, d, h))
    _check_int8_dims(op, e, d, h)
    code = _check_int8_bias(op, mlp1_bias, (e, 2 * h))
    if _check_int8_bias(op, mlp2_bias, (e, d)) != code:
        raise TypeError(f"{op} takes both biases in one dtype, got {mlp1_bias.dtype} and {mlp2_bias.dtype}")
    if not swiglu_limit >= 0:
        raise ValueError(f"{op} expects a clamp limit of at least 0, got {swiglu_limit}")
    x, qmlp1, qmlp2 = map(_ready, (x, qmlp1, qmlp2))
    smlp1, smlp2, b1, b2 = (t.contiguous() for t in (smlp1, smlp2, mlp1_bias, mlp2_bias))
    ws_bytes = _int8_layer_workspace_bytes(r, e, d, h)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    y = torch.empty_like(x)
    _int8_launch(here, "moe_int8_oss", x, x.data_ptr(), qmlp1.data_ptr(), smlp1.data_ptr(), b1.data_ptr(), qmlp2.data_ptr(),
                 smlp2.data_ptr(), b2.data_ptr(), code, counts.data_ptr(), r, e, d, h, float(swiglu_limit), ws.data_ptr(), ws_bytes,
                 y.data_ptr())
    return y


@torch.library.register_fake("moe_mi355x_int8_bare::grouped_swiglu_oss_int8", lib=_I8_BARE)
def _(x, qmlp1, smlp1, mlp1_bias, qmlp2, smlp2, mlp2_bias, num_tokens_per_expert, swiglu_limit):
    return x.new_empty(x.shape)


@_inference_op(_grouped_swiglu_oss_int8, _I8)
def grouped_swiglu_oss_int8(
    x: Tensor, qmlp1: Tensor, smlp1: Tensor, mlp1_bias: Tensor, qmlp2: Tensor, smlp2: Tensor, mlp2_bias: Tensor,
    num_tokens_per_expert: Tensor, swiglu_limit: float,
) -> Tensor:
    """grouped_swiglu_int8 for gpt-oss's experts (gpt_oss/moe.py:43-122): mlp1 [E, 2H, D] (glu row 2j,
    linear row 2j + 1) and mlp2 [E, D, H] in codes, biases [E, 2H] and [E, D], both in bf16 or both
    in fp32; biases, clamps and activation in fp32 between the products."""
    _no_int8_gradients("grouped_swiglu_oss_int8", x, smlp1, mlp1_bias, smlp2, mlp2_bias)
    return _grouped_swiglu_oss_int8(x, qmlp1, smlp1, mlp1_bias, qmlp2, smlp2, mlp2_bias, num_tokens_per_expert, swiglu_limit)


# ---------------------------------------------------------------------------
# the routed half of MoE.forward with fp8 experts and the score applied before
# them, the permute folded into the token quantizers
# ---------------------------------------------------------------------------
def _aligned(src: Tensor) -> Tensor:
    return src.clone() if src.data_ptr() % 16 else src  # the gathering kernels read rows in 16-byte pieces


def _quant_rows_groupamax_gather(src: Tensor, token_idx: Tensor, row_scale: Tensor | None, counts: Tensor,
                                 e: int) -> tuple[Tensor, Tensor, Tensor]:
    """_quant_rows_groupamax of the routed rows src[token_idx] (* row_scale, rounded
    to bf16), read from src [N, C] in place."""
    src = _aligned(src)
    r, c = token_idx.shape[0], src.shape[1]
    q = torch.empty(r, c, dtype=FP8, device=src.device)
    sc = torch.empty(r, dtype=torch.float32, device=src.device)
    amax = torch.zeros(e, c, dtype=torch.float32, device=src.device)
    call("moe_fp8_quant_rows_groupamax_gather", ptr(src), src.shape[0], ptr(token_idx), ptr(row_scale), ptr(counts),
         r, e, c, ptr(q), ptr(sc), ptr(amax), stream_of(src))
    return q, sc, amax


def _quant_tokens_t_gather(src: Tensor, token_idx: Tensor, row_scale: Tensor | None, counts: Tensor, e: int,
                           rpad: int, amax: Tensor) -> tuple[Tensor, Tensor]:
    """_quant_tokens_t (from the groups' known amax) of the routed rows
    src[token_idx] (* row_scale, rounded to bf16), read from src in place."""
    src = _aligned(src)
    r, c = token_idx.shape[0], src.shape[1]
    q = torch.empty(c, rpad, dtype=FP8, device=src.device)
    sc = torch.empty(e, c, dtype=torch.float32, device=src.device)
    call("moe_fp8_quant_tokens_t_amax_gather", ptr(src), src.shape[0], ptr(token_idx), ptr(row_scale), ptr(amax),
         ptr(counts), r, e, c, rpad, ptr(q), ptr(sc), stream_of(src))
    return q, sc


@torch.library.custom_op("moe_mi355x::moe_core_fp8", mutates_args=())
def moe_core_fp8(
    x: Tensor, shared_out: Tensor | None, token_idx: Tensor, scores_sorted: Tensor, slot_pos: Tensor,
    tok_pos: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor,
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """out = combine(shared_out, experts(x[token_idx] * score)) with fp8 experts
    (moe.py:440-470 with score_before_experts; the ops of permute,
    grouped_swiglu_fp8 and combine): the routed rows are quantized straight from x
    (moe_fp8_quant_rows_groupamax_gather), so no routed copy of x is written, and
    in the backward the routed gradient and the routed x are quantized straight
    from the output's gradient and from x. Returns (out, g, u, h, then the column
    amax of w1, w3, w2, of the routed x and of h per token group)."""
    require_gpu(x, shared_out, token_idx, scores_sorted, slot_pos, tok_pos, w1, w2, w3, num_tokens_per_expert)
    _check_bf16("moe_core_fp8", x=x, w1=w1, w2=w2, w3=w3)
    x, w1, w2, w3 = x.contiguous(), w1.contiguous(), w2.contiguous(), w3.contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    tidx = token_idx.to(torch.int64).contiguous()
    sc = scores_sorted.float().contiguous()
    qx, sx, amx = _quant_rows_groupamax_gather(x, tidx, sc, counts, w1.shape[0])
    y, g, u, h, am1, am3, am2, amh = _fp8_experts_forward(qx, sx, w1, w2, w3, counts)
    out = combine(shared_out, y, slot_pos, tok_pos, None)
    return out, g, u, h, am1, am3, am2, amx, amh


@moe_core_fp8.register_fake
def _(x, shared_out, token_idx, scores_sorted, slot_pos, tok_pos, w1, w2, w3, num_tokens_per_expert):
    n, d = x.shape
    r = token_idx.shape[0]
    e, h_dim, _ = w1.shape
    f32 = lambda *shape: x.new_empty(*shape, dtype=torch.float32)  # noqa: E731
    return (x.new_empty(n, d), x.new_empty(r, h_dim), x.new_empty(r, h_dim), x.new_empty(r, h_dim),
            f32(*_amax_shape(e, d)), f32(*_amax_shape(e, d)), f32(*_amax_shape(e, h_dim)), f32(e, d),
            f32(*_amax_shape(e, h_dim)))


@torch.library.custom_op("moe_mi355x::moe_core_fp8_backward", mutates_args=())
def moe_core_fp8_backward(
    grad_out: Tensor, x: Tensor, token_idx: Tensor, scores_sorted: Tensor, tok_pos: Tensor, w1: Tensor,
    w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor, g: Tensor, u: Tensor, h: Tensor, amax_w1: Tensor,
    amax_w3: Tensor, amax_w2: Tensor, amax_x: Tensor, amax_h: Tensor,
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(grad_x, grad_scores_sorted, dw1, dw2, dw3) of moe_core_fp8's out; the
    shared output's gradient is grad_out itself (the combine adds it once)."""
    require_gpu(grad_out, x, token_idx, scores_sorted, tok_pos, w1, w2, w3, num_tokens_per_expert, g, u, h)
    go = grad_out.to(torch.bfloat16).contiguous()
    x = x.contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    tidx = token_idx.to(torch.int64).contiguous()
    sc = scores_sorted.float().contiguous()
    e = w1.shape[0]
    qdy, sdy, amdy = _quant_rows_groupamax_gather(go, tidx, None, counts, e)
    dx_routed, dw1, dw2, dw3 = _fp8_experts_backward(
        qdy, sdy, w1, w2, w3, counts, g, u, h, amax_w1, amax_w3, amax_w2, amax_h,
        lambda rpad: _quant_tokens_t_gather(x, tidx, sc, counts, e, rpad, amax_x),
        lambda rpad: _quant_tokens_t_gather(go, tidx, None, counts, e, rpad, amdy))
    grad_x, grad_s = permute_backward(dx_routed, x, tok_pos, scores_sorted, PERMUTE_BWD_ROUND_EACH)
    return grad_x, grad_s, dw1, dw2, dw3


@moe_core_fp8_backward.register_fake
def _(grad_out, x, token_idx, scores_sorted, tok_pos, w1, w2, w3, num_tokens_per_expert, *saved):
    r = token_idx.shape[0]
    return (x.new_empty(x.shape), x.new_empty(r, dtype=torch.float32), torch.empty_like(w1), torch.empty_like(w2),
            torch.empty_like(w3))


def _core_fp8_setup(ctx, inputs, output):
    x, shared_out, token_idx, scores_sorted, _slot_pos, tok_pos, w1, w2, w3, counts = inputs
    _out, g, u, h, *amax = output
    ctx.save_for_backward(x, token_idx, scores_sorted, tok_pos, w1, w2, w3, counts, g, u, h, *amax)
    ctx.has_shared = shared_out is not None
    ctx.shared_dtype = shared_out.dtype if shared_out is not None else None
    ctx.mark_non_differentiable(g, u, h, *amax)
    ctx.set_materialize_grads(False)


def _core_fp8_bwd(ctx, grad_out, *_unused):
    if grad_out is None:
        return (None,) * 10
    x, token_idx, scores_sorted, tok_pos, w1, w2, w3, counts, g, u, h, *amax = ctx.saved_tensors
    grad_x, grad_s, dw1, dw2, dw3 = moe_core_fp8_backward(grad_out, x, token_idx, scores_sorted, tok_pos, w1, w2,
                                                          w3, counts, g, u, h, *amax)
    grad_shared = grad_out.to(ctx.shared_dtype) if ctx.has_shared else None
    return grad_x, grad_shared, None, grad_s, None, None, dw1, dw2, dw3, None


moe_core_fp8.register_autograd(_core_fp8_bwd, setup_context=_core_fp8_setup)


# ---------------------------------------------------------------------------
# the routed half of MoE.forward with MXFP8 experts and the score applied before
# them, the permute folded into the token quantizer
# ---------------------------------------------------------------------------
def _mx_dual_tokens_gather(src: Tensor, token_idx: Tensor, row_scale: Tensor | None, counts: Tensor, e: int,
                           rpad: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """_mx_dual_tokens of the routed rows src[token_idx] (* row_scale, rounded to
    bf16), read from src [N, C] in place."""
    src = _aligned(src)
    r = token_idx.shape[0]
    c = src.shape[1]
    qr = torch.empty(r, c, dtype=FP8, device=src.device)
    sr = torch.empty(r, c // MX_BLOCK, dtype=torch.uint8, device=src.device)
    qt = torch.empty(c, rpad, dtype=FP8, device=src.device)
    st = torch.empty(rpad // MX_BLOCK, c, dtype=torch.uint8, device=src.device)
    call("moe_mxfp8_quant_dual_tokens_gather", ptr(src), src.shape[0], ptr(token_idx), ptr(row_scale), ptr(counts),
         r, e, c, rpad, ptr(qr), ptr(sr), ptr(qt), ptr(st), stream_of(src))
    return qr, sr, qt, st


@torch.library.custom_op("moe_mi355x::moe_core_mxfp8", mutates_args=())
def moe_core_mxfp8(
    x: Tensor, shared_out: Tensor | None, token_idx: Tensor, scores_sorted: Tensor, slot_pos: Tensor,
    tok_pos: Tensor, w1: Tensor, w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor,
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """out = combine(shared_out, experts(x[token_idx] * score)) with MXFP8 experts
    (moe.py:440-470 with score_before_experts; the ops of permute,
    grouped_swiglu_mxfp8 and combine): the routed rows are quantized straight from
    x (moe_mxfp8_quant_dual_tokens_gather), so no routed copy of x is written, and
    in the backward the routed gradient is quantized straight from the output's
    gradient. Returns (out, g, u, h, then the forward's quantized layouts the
    backward reuses)."""
    require_gpu(x, shared_out, token_idx, scores_sorted, slot_pos, tok_pos, w1, w2, w3, num_tokens_per_expert)
    _check_bf16("moe_core_mxfp8", x=x, w1=w1, w2=w2, w3=w3)
    x, w1, w2, w3 = x.contiguous(), w1.contiguous(), w2.contiguous(), w3.contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    tidx = token_idx.to(torch.int64).contiguous()
    sc = scores_sorted.float().contiguous()
    r = tidx.shape[0]
    d = x.shape[1]
    e, h_dim, _ = w1.shape
    s = stream_of(x)
    rpad = _mx_padded_rows(r, e)
    qx, sx, qxt, sxt = _mx_dual_tokens_gather(x, tidx, sc, counts, e, rpad)
    qw1, sw1, qw3, sw3, qw2, sw2, qw2t, sw2t, qw13t, sw13t = _mx_weights(w1, w2, w3, True)
    g = x.new_empty(r, h_dim)
    u = x.new_empty(r, h_dim)
    h = x.new_empty(r, h_dim)
    call("moe_mxfp8_gemm_gate_up", ptr(qx), ptr(sx), ptr(qw1), ptr(sw1), ptr(qw3), ptr(sw3), ptr(counts), r, e, d,
         h_dim, ptr(g), ptr(u), ptr(h), s)
    qh, sh, qht, sht = _mx_dual_tokens(h, counts, e, rpad)
    y = x.new_empty(r, d)
    call("moe_mxfp8_gemm_down", ptr(qh), ptr(sh), ptr(qw2), ptr(sw2), ptr(counts), r, e, d, h_dim, ptr(y), s)
    out = combine(shared_out, y, slot_pos, tok_pos, None)
    return out, g, u, h, qxt, sxt, qht, sht, qw2t, sw2t, qw13t, sw13t


@moe_core_mxfp8.register_fake
def _(x, shared_out, token_idx, scores_sorted, slot_pos, tok_pos, w1, w2, w3, num_tokens_per_expert):
    n, d = x.shape
    r = token_idx.shape[0]
    e, h_dim, _ = w1.shape
    u8 = lambda *shape: x.new_empty(*shape, dtype=torch.uint8)  # noqa: E731
    rpad = (r + e * 127 + 127) // 128 * 128  # _mx_padded_rows
    return (x.new_empty(n, d), x.new_empty(r, h_dim), x.new_empty(r, h_dim), x.new_empty(r, h_dim),
            u8(d, rpad), u8(rpad // 32, d), u8(h_dim, rpad), u8(rpad // 32, h_dim),
            u8(e, h_dim, d), u8(e, h_dim, d // 32), u8(e, d, 2 * h_dim), u8(e, d, 2 * h_dim // 32))


@torch.library.custom_op("moe_mi355x::moe_core_mxfp8_backward", mutates_args=())
def moe_core_mxfp8_backward(
    grad_out: Tensor, x: Tensor, token_idx: Tensor, scores_sorted: Tensor, tok_pos: Tensor, w1: Tensor,
    w2: Tensor, w3: Tensor, num_tokens_per_expert: Tensor, g: Tensor, u: Tensor, h: Tensor, qxt: Tensor,
    sxt: Tensor, qht: Tensor, sht: Tensor, qw2t: Tensor, sw2t: Tensor, qw13t: Tensor, sw13t: Tensor,
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(grad_x, grad_scores_sorted, dw1, dw2, dw3) of moe_core_mxfp8's out; the
    shared output's gradient is grad_out itself (the combine adds it once)."""
    require_gpu(grad_out, x, token_idx, scores_sorted, tok_pos, w1, w2, w3, num_tokens_per_expert, g, u, h)
    go = grad_out.to(torch.bfloat16).contiguous()
    counts = num_tokens_per_expert.to(torch.int64).contiguous()
    tidx = token_idx.to(torch.int64).contiguous()
    r = tidx.shape[0]
    d = x.shape[1]
    e = w1.shape[0]
    rpad = _mx_padded_rows(r, e)
    qdy = _mx_dual_tokens_gather(go, tidx, None, counts, e, rpad)
    dx_routed, dw1, dw2, dw3 = _mx_experts_backward(qdy, r, d, w1, w2, w3, counts, g, u, h, qxt, sxt, qht, sht,
                                                    qw2t, sw2t, qw13t, sw13t, rpad)
    grad_x, grad_s = permute_backward(dx_routed, x, tok_pos, scores_sorted, PERMUTE_BWD_ROUND_EACH)
    return grad_x, grad_s, dw1, dw2, dw3


@moe_core_mxfp8_backward.register_fake
def _(grad_out, x, token_idx, scores_sorted, tok_pos, w1, w2, w3, num_tokens_per_expert, *saved):
    r = token_idx.shape[0]
    return (x.new_empty(x.shape), x.new_empty(r, dtype=torch.float32), torch.empty_like(w1), torch.empty_like(w2),
            torch.empty_like(w3))


def _core_mx_setup(ctx, inputs, output):
    x, shared_out, token_idx, scores_sorted, _slot_pos, tok_pos, w1, w2, w3, counts = inputs
    _out, g, u, h, *quantized = output
    ctx.save_for_backward(x, token_idx, scores_sorted, tok_pos, w1, w2, w3, counts, g, u, h, *quantized)
    ctx.has_shared = shared_out is not None
    ctx.shared_dtype = shared_out.dtype if shared_out is not None else None
    ctx.mark_non_differentiable(g, u, h, *quantized)
    ctx.set_materialize_grads(False)


def _core_mx_bwd(ctx, grad_out, *_unused):
    if grad_out is None:
        return (None,) * 10
    x, token_idx, scores_sorted, tok_pos, w1, w2, w3, counts, g, u, h, *quantized = ctx.saved_tensors
    grad_x, grad_s, dw1, dw2, dw3 = moe_core_mxfp8_backward(grad_out, x, token_idx, scores_sorted, tok_pos, w1, w2,
                                                            w3, counts, g, u, h, *quantized)
    grad_shared = grad_out.to(ctx.shared_dtype) if ctx.has_shared else None
    return grad_x, grad_shared, None, grad_s, None, None, dw1, dw2, dw3, None


moe_core_mxfp8.register_autograd(_core_mx_bwd, setup_context=_core_mx_setup)


# ---------------------------------------------------------------------------
# row gather / scatter by an index (expert-parallel permute and unpermute)
# ---------------------------------------------------------------------------
@torch.library.custom_op("moe_mi355x::gather_rows", mutates_args=())
def gather_rows(src: Tensor, idx: Tensor) -> Tensor:
    """dst = src[idx, :] (expert_parallel.py:70-74)."""
    require_gpu(src, idx)
    s = src.contiguous()
    ix = idx.to(torch.int64).contiguous()
    n, d = ix.shape[0], s.shape[1]
    out = s.new_empty(n, d)
    call("moe_gather_rows", ptr(s), s.shape[0], ptr(ix), n, d, _dtype_code(s), ptr(out), stream_of(s))
    return out


@gather_rows.register_fake
def _(src, idx):
    return src.new_empty(idx.shape[0], src.shape[1])


@torch.library.custom_op("moe_mi355x::scatter_rows", mutates_args=())
def scatter_rows(src: Tensor, idx: Tensor, n_rows: int) -> Tensor:
    """dst = empty(n_rows, d); dst[idx, :] = src (expert_parallel.py:77-80). Rows of
    dst that idx does not name are left uninitialised, as in the reference."""
    require_gpu(src, idx)
    s = src.contiguous()
    ix = idx.to(torch.int64).contiguous()
    out = s.new_empty(n_rows, s.shape[1])
    call("moe_scatter_rows", ptr(s), ptr(ix), ix.shape[0], s.shape[1], _dtype_code(s), ptr(out), n_rows,
         stream_of(s))
    return out


@scatter_rows.register_fake
def _(src, idx, n_rows):
    return src.new_empty(n_rows, src.shape[1])


def _rows_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[1])
    ctx.n_src = inputs[0].shape[0]


def _gather_rows_bwd(ctx, g):
    # a permutation: every source row receives exactly one gradient row
    (idx,) = ctx.saved_tensors
    return scatter_rows(g, idx, ctx.n_src), None


def _scatter_rows_bwd(ctx, g):
    (idx,) = ctx.saved_tensors
    return gather_rows(g, idx), None, None


gather_rows.register_autograd(_gather_rows_bwd, setup_context=_rows_setup)
scatter_rows.register_autograd(_scatter_rows_bwd, setup_context=_rows_setup)
