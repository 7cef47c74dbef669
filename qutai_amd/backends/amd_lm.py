"""Decoder-LM kernels of the amd device (sibling of src/qutai/backends/cuda_lm.py).

Same names and argument meaning as the reference LM backend for the
contraction path: ``gemm`` (cuda_lm.py:31-55), ``routing`` (:368-449),
``route_gather`` / ``route_gather_backward`` (:471-502), ``combine`` /
``combine_backward`` (:505-581), ``silu`` products, ``take``.  Additions that
the MI355X design needs: ``route_gather_all`` and ``combine_all`` (one launch
for every expert), ``grouped_gemm`` and ``moe_experts_forward`` (the expert
projections as grouped GEMMs whose per-expert row ranges stay in device
memory, so no host synchronisation sizes them).
"""
from __future__ import annotations

from array import array
from itertools import compress, islice
from operator import ne
from random import Random

from . import amd
from .amd import _TYPES, AMDStorage, code
from .amd_runtime import get_runtime
from ..core.grad import DeferredGradient


def normal(size, mean=0.0, std=1.0, *, seed=None, dtype="float32"):
    """Host-drawn N(mean, std) values (Random(seed).gauss, as the CPU path
    draws them: src/qutai/backends/cpu_lm.py:6-8), uploaded once."""
    random = Random(seed)
    return amd.storage(array("f", (random.gauss(mean, std) for _ in range(size))), dtype=dtype)


def gemm(a, b, rows, inner, cols, *, transpose_left=False, transpose_right=False, out_dtype=None, out=None,
         accumulate=False):
    """LM GEMM without batch/strides (src/qutai/backends/cuda_lm.py:31-55)."""
    return amd.gemm(a, b, rows, inner, cols, transpose_left=transpose_left, transpose_right=transpose_right,
                    out_dtype=out_dtype, out=out, accumulate=accumulate)


def take(values, start, size):
    return amd.take(values, start, size)


def silu_mul(gate: AMDStorage, up: AMDStorage) -> AMDStorage:
    """silu(gate) * up with the reference's per-op rounding."""
    if (gate.dtype, gate.size) != (up.dtype, up.size):
        raise ValueError("silu_mul needs operands of equal dtype and size")
    out = AMDStorage(gate.size, gate.dtype)
    if gate.size:
        out.runtime.call("qutai_amd_silu_mul", gate.ptr, up.ptr, out.ptr, gate.size, code(gate.dtype))
    return out


def silu_mul_backward(gradient, gate, up):
    dgate, dup = AMDStorage(gate.size, gate.dtype), AMDStorage(up.size, up.dtype)
    if gate.size:
        dgate.runtime.call("qutai_amd_silu_mul_backward", gradient.ptr, gate.ptr, up.ptr, dgate.ptr, dup.ptr,
                           gate.size, code(gate.dtype))
    return dgate, dup


def _route_workspace_bytes(runtime, rows, experts, top_k):
    """Workspace of the chunked routing path (0: the per-expert pack)."""
    return runtime.lib.qutai_amd_route_workspace_size(rows, experts, top_k)


def routing(scores, rows, experts, top_k, *, download_counts=True):
    """Router softmax, top-k selection and stable per-expert packing.

    Returns the dict of ``cuda_lm.routing`` (cuda_lm.py:436-449): probs,
    weights, indices, counts, ids, slots, locations, utilization, aux, rows,
    experts, top_k, capacity; plus ``offsets`` ([experts+1], device) and
    ``order`` (token ids expert-major, device) used by the one-launch gather
    and the grouped GEMMs.  ``counts`` is a host tuple (one device read, as
    in the reference) unless ``download_counts`` is False.
    """
    if scores.dtype == "bfloat16":
        scores = amd.from_storage(scores, dtype="float32")
    if scores.dtype != "float32":
        raise ValueError("amd routing takes float32 or bfloat16 router scores")
    if experts <= 0 or not 0 < top_k <= experts or scores.size != rows * experts:
        raise ValueError("routing needs 0 < top_k <= experts and rows * experts scores")
    capacity = rows * top_k
    probs = AMDStorage(rows * experts, "float32")
    weights = AMDStorage(capacity, "float32")
    indices = AMDStorage(capacity, "int64")
    counts = AMDStorage(experts, "int64")
    ids = AMDStorage(experts * capacity, "int64")
    slots = AMDStorage(experts * capacity, "int64")
    locations = AMDStorage(capacity, "int64")
    offsets = AMDStorage(experts + 1, "int64")
    order = AMDStorage(capacity, "int64")
    utilization = AMDStorage(experts, "float32")
    aux = AMDStorage(1, "float32")
    runtime = get_runtime()
    need = _route_workspace_bytes(runtime, rows, experts, top_k)
    workspace = AMDStorage((need + 3) // 4, "float32") if need else None
    runtime.call("qutai_amd_route", scores.ptr, probs.ptr, weights.ptr, indices.ptr, counts.ptr, ids.ptr, slots.ptr,
                 locations.ptr, offsets.ptr, order.ptr, utilization.ptr, aux.ptr, rows, experts, top_k,
                 workspace.ptr if workspace else None, need)
    host_counts = tuple(counts.to_array().tolist()) if download_counts else None
    return dict(probs=probs, weights=weights, indices=indices, counts=host_counts, count_buffer=counts, ids=ids,
                slots=slots, locations=locations, offsets=offsets, order=order, utilization=utilization, aux=aux,
                rows=rows, experts=experts, top_k=top_k, capacity=capacity)


def _host_offsets(route):
    counts = route["counts"]
    if counts is None:
        raise ValueError("per-expert calls need the host counts (routing(..., download_counts=True))")
    starts = [0]
    for count in counts:
        starts.append(starts[-1] + count)
    return starts


def route_gather(values, route, expert, width):
    """Rows of one expert, in token order (cuda_lm.py:471-485)."""
    start = _host_offsets(route)[expert]
    count = route["counts"][expert]
    result = AMDStorage(count * width, values.dtype)
    if count * width:
        result.runtime.call("qutai_amd_route_gather", values.ptr, route["order"].ptr + 8 * start, result.ptr, count,
                            width, 0, code(values.dtype))
    return result


def route_gather_backward(gradient, route, expert, width):
    """Scatter one expert's row gradients back to token rows (cuda_lm.py:488-502)."""
    start = _host_offsets(route)[expert]
    count = route["counts"][expert]
    result = amd.full(route["rows"] * width, 0.0, dtype=gradient.dtype)
    if count * width:
        result.runtime.call("qutai_amd_route_gather", gradient.ptr, route["order"].ptr + 8 * start, result.ptr,
                            count, width, 1, code(gradient.dtype))
    return result


def route_gather_all(values, route, width):
    """All experts' token rows in one expert-major block [rows*top_k, width]."""
    total = route["capacity"]
    result = AMDStorage(total * width, values.dtype)
    if total * width:
        result.runtime.call("qutai_amd_route_gather", values.ptr, route["order"].ptr, result.ptr, total, width, 0,
                            code(values.dtype))
    return result


def combine_all(expert_rows, route, width):
    """y[row] = sum_slot weight * expert output row, from the expert-major
    block produced by the grouped GEMMs (one launch, fp32 sum, one rounding)."""
    result = AMDStorage(route["rows"] * width, expert_rows.dtype)
    if result.size:
        result.runtime.call("qutai_amd_combine", expert_rows.ptr, route["weights"].ptr, route["indices"].ptr,
                            route["locations"].ptr, route["offsets"].ptr, result.ptr, route["rows"], width,
                            route["top_k"], code(expert_rows.dtype), code(expert_rows.dtype))
    return result


def combine(outputs, weights, route, width):
    """Reference-shaped combine over a list of (expert, rows) outputs
    (cuda_lm.py:505-541): the rows are laid out expert-major and combined
    in one launch."""
    if weights is not route["weights"]:
        route = dict(route, weights=weights)
    dtype = outputs[0][1].dtype if outputs else "float32"
    block = AMDStorage(route["capacity"] * width, dtype)
    starts = _host_offsets(route)
    item = 2 if dtype == "bfloat16" else 4
    for expert, values in outputs:
        if values.size:
            block.runtime.copy(block.ptr + starts[expert] * width * item, values.ptr, values.nbytes)
    return combine_all(block, route, width)


def grouped_gemm(rows_block, weight_stack, route, inner, cols, *, out_dtype="bfloat16", transpose_right=True,
                 out=None, accumulate=False, gather=False):
    """out[offsets[e]:offsets[e+1]] (+)= rows_block[offsets[e]:offsets[e+1]] @ op(W_e)
    for every expert in one launch, the row ranges read on the device.  With
    ``transpose_right`` W_e = weight_stack[e] is stored (cols, inner) and used
    transposed (the forward X W^T); without, it is stored (inner, cols) (the
    backward dY W).  With ``gather`` rows_block is the token matrix
    [rows][inner] and the expert-major rows are read through ``order``
    inside the GEMM (no gathered copy)."""
    experts = route["experts"]
    if weight_stack.size != experts * cols * inner or rows_block.dtype != weight_stack.dtype:
        raise ValueError("grouped_gemm needs [experts] weights of cols*inner values in the rows' dtype")
    source = route["rows"] if gather else route["capacity"]
    if rows_block.size != source * inner:
        raise ValueError("grouped_gemm rows do not match the route (rows x inner, or capacity x inner)")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = AMDStorage(route["capacity"] * cols, out_dtype)
    elif out.dtype != out_dtype or out.size != route["capacity"] * cols:
        raise ValueError("out must hold capacity x cols values of out_dtype")
    if out.size:
        out.runtime.call("qutai_amd_gemm_grouped", rows_block.ptr, weight_stack.ptr, out.ptr, route["offsets"].ptr,
                         experts, route["capacity"], inner, cols, cols * inner, int(transpose_right),
                         code(rows_block.dtype), code(out_dtype), int(accumulate),
                         route["order"].ptr if gather else None, source if gather else 0, mfma=True)
    return out


def grouped_gemm_pair(rows_block, rows_tail, weight_stack, weight_tail, route, inner, cols, *,
                      out_dtype="float32", transpose_right=False):
    """out[offsets[e]:offsets[e+1]] = rows_block[..] @ op(W_e) + rows_tail[..] @ op(Wtail_e)
    in one launch and one accumulator (qutai_amd_gemm_grouped_pair): the two
    products of grouped_gemm summed over K = 2 * inner without an fp32
    partial in between; inner a multiple of 64."""
    experts = route["experts"]
    for block, stack in ((rows_block, weight_stack), (rows_tail, weight_tail)):
        if stack.size != experts * cols * inner or block.dtype != stack.dtype or block.dtype != rows_block.dtype:
            raise ValueError("grouped_gemm_pair needs [experts] weights of cols*inner values in the rows' dtype")
        if block.size != route["capacity"] * inner:
            raise ValueError("grouped_gemm_pair rows must be capacity x inner")
    if inner % 64:
        raise ValueError("grouped_gemm_pair joins its two halves at a multiple of 64")
    out = AMDStorage(route["capacity"] * cols, out_dtype)
    if out.size:
        out.runtime.call("qutai_amd_gemm_grouped_pair", rows_block.ptr, rows_tail.ptr, weight_stack.ptr,
                         weight_tail.ptr, out.ptr, route["offsets"].ptr, experts, route["capacity"], inner, cols,
                         cols * inner, int(transpose_right), code(rows_block.dtype), code(out_dtype), 0, mfma=True)
    return out


def swiglu_gemm(rows_block, w_gate, w_up, rows, inner, hidden, *, route=None, save=False, gather=False):
    """silu(rows_block @ W_gate^T) * (rows_block @ W_up^T) in one bf16 GEMM
    (qutai_amd_gemm_swiglu), with the unfused form's roundings.  With
    ``route`` the rows are grouped by expert and W_* are [experts][hidden][inner]
    stacks; without, one [hidden][inner] weight pair and ``rows`` rows.  With
    ``gather`` (grouped only) rows_block is the token matrix and the routed
    rows are read through ``order`` inside the GEMM.  With ``save`` the bf16
    gate and up products are returned too (for the backward): (act, gate, up)."""
    if route is not None:
        rows, groups = route["capacity"], route["experts"]
    elif gather:
        raise ValueError("swiglu_gemm gathers rows only for a route")
    else:
        groups = 1
    source = route["rows"] if gather else rows
    if rows_block.dtype != "bfloat16" or {w_gate.dtype, w_up.dtype} != {"bfloat16"}:
        raise ValueError("swiglu_gemm runs bf16 operands")
    if rows_block.size != source * inner or w_gate.size != groups * hidden * inner or w_up.size != w_gate.size:
        raise ValueError("swiglu_gemm operand sizes do not match rows, inner and hidden")
    act = AMDStorage(rows * hidden, "bfloat16")
    gate = AMDStorage(rows * hidden, "bfloat16") if save else None
    up = AMDStorage(rows * hidden, "bfloat16") if save else None
    if act.size:
        act.runtime.call("qutai_amd_gemm_swiglu", rows_block.ptr, w_gate.ptr, w_up.ptr, act.ptr,
                         gate.ptr if save else None, up.ptr if save else None,
                         route["offsets"].ptr if route is not None else None, groups, rows, inner, hidden,
                         hidden * inner, code("bfloat16"), route["order"].ptr if gather else None,
                         source if gather else 0, mfma=True)
    return (act, gate, up) if save else act


def grouped_gemm_k(a_block, b_block, route, rows, cols, *, out_dtype="float32", gather=False):
    """out[e] = A_e^T B_e for every expert, A_e / B_e the expert-major routed
    rows of a_block ([capacity][rows]) and b_block ([capacity][cols]): the
    per-expert weight gradients in one launch (an expert with no rows gets
    zeros).  With ``gather`` b_block is the token matrix ([route rows][cols])
    and B_e's rows are read through the route's ``order`` inside the GEMM."""
    experts = route["experts"]
    b_rows = route["rows"] if gather else route["capacity"]
    if a_block.dtype != b_block.dtype or a_block.size != route["capacity"] * rows or b_block.size != b_rows * cols:
        raise ValueError("grouped_gemm_k needs [capacity][rows] and [capacity][cols] (gathered: [tokens][cols]) "
                         "blocks of one dtype")
    out = AMDStorage(experts * rows * cols, out_dtype)
    if out.size:
        out.runtime.call("qutai_amd_gemm_grouped_k", a_block.ptr, b_block.ptr, out.ptr, route["offsets"].ptr, experts,
                         rows, cols, route["capacity"], code(a_block.dtype), code(out_dtype), 0,
                         route["order"].ptr if gather else None, b_rows if gather else 0, mfma=True)
    return out


def _as_dtype(values, dtype):
    return values if values.dtype == dtype else amd.from_storage(values, dtype=dtype)


def repitch(values, batches, rows, cols, new_rows, new_cols):
    """[batches][rows][cols] -> [batches][new_rows][new_cols], zero padded or cropped."""
    if values.size != batches * rows * cols:
        raise ValueError("repitch source size does not match its shape")
    out = AMDStorage(batches * new_rows * new_cols, values.dtype)
    if out.size:
        out.runtime.call("qutai_amd_repitch", values.ptr, out.ptr, batches, rows, cols, new_rows, new_cols,
                         code(values.dtype))
    return out


def _pad8(n):
    return (n + 7) // 8 * 8


def _rows_through_order(token_bytes, *, dtype):
    """Whether the expert products read the routed token rows through the
    route's ``order`` inside the grouped GEMMs (the forward's gate/up and,
    in training, the backward's dW_gate / dW_up) instead of copying them:
    bf16 or fp32 tokens and a token matrix below 2 GiB (the GEMMs address it
    with 32-bit byte offsets of one buffer descriptor)."""
    return dtype in ("bfloat16", "float32") and token_bytes < (1 << 31)


def moe_experts_forward(x, route, w_gate, w_up, w_down, width, hidden, *, save=False):
    """Expert SwiGLU for every routed (token, slot): gather, grouped gate/up
    and silu(gate) * up (one fused grouped GEMM for bf16, same roundings),
    grouped down, weighted combine (lm/layers.py:395-399).
    Weights of another dtype than x (fp32 master weights, bf16 activations)
    are rounded to x's dtype for the products, as the reference's mixed GEMM
    does.  Widths that are not multiples of 8 run zero padded to the next
    multiple (padded weight rows and columns are zero, so the padded outputs
    are zero and the cropped result is exact).  With ``save`` the
    intermediates for ``moe_experts_backward`` are returned too."""
    wp, hp = _pad8(width), _pad8(hidden)
    experts = route["experts"]
    wg, wu, wd = (_as_dtype(w, x.dtype) for w in (w_gate, w_up, w_down))
    fused = _rows_through_order(x.nbytes, dtype=x.dtype)
    rows = x if fused else route_gather_all(x, route, width)
    if (wp, hp) != (width, hidden):
        wg, wu = (repitch(w, experts, hidden, width, hp, wp) for w in (wg, wu))
        wd = repitch(wd, experts, width, hidden, wp, hp)
        rows = repitch(rows, 1, route["rows"] if fused else route["capacity"], width,
                       route["rows"] if fused else route["capacity"], wp)
    if x.dtype == "bfloat16" and save:
        act, gate, up = swiglu_gemm(rows, wg, wu, 0, wp, hp, route=route, save=True, gather=fused)
    elif x.dtype == "bfloat16":
        act, gate, up = swiglu_gemm(rows, wg, wu, 0, wp, hp, route=route, gather=fused), None, None
    else:
        gate = grouped_gemm(rows, wg, route, wp, hp, out_dtype=x.dtype, gather=fused)
        up = grouped_gemm(rows, wu, route, wp, hp, out_dtype=x.dtype, gather=fused)
        act = silu_mul(gate, up)
    down = grouped_gemm(act, wd, route, hp, wp, out_dtype=x.dtype)
    if wp != width:
        down = repitch(down, 1, route["capacity"], wp, route["capacity"], width)
    y = combine_all(down, route, width)
    if not save:
        return y
    # rows: the (padded) token matrix when the products read it through the
    # route's order (gathered), else the expert-major routed copy
    return y, dict(rows=rows, gathered=fused, gate=gate, up=up, act=act, down=down, w_gate=wg, w_up=wu, w_down=wd)


def combine_backward_all(gradient, expert_rows, route, width):
    """(d expert rows [capacity][width], d weights [rows*top_k] fp32) of
    combine_all, one launch for every (token, slot)."""
    d_rows = AMDStorage(expert_rows.size, expert_rows.dtype)
    d_weights = AMDStorage(route["capacity"], "float32")
    if route["capacity"]:
        d_rows.runtime.call("qutai_amd_combine_backward", gradient.ptr, expert_rows.ptr, route["weights"].ptr,
                            route["indices"].ptr, route["locations"].ptr, route["offsets"].ptr, d_rows.ptr,
                            d_weights.ptr, route["rows"], width, route["top_k"], code(expert_rows.dtype))
    return d_rows, d_weights


def combine_backward(gradient, outputs, weights, route, width):
    """Reference-shaped combine backward (cuda_lm.py:544-581): per-expert row
    gradients in the order of ``outputs``, then the weight gradient."""
    if weights is not route["weights"]:
        route = dict(route, weights=weights)
    dtype = outputs[0][1].dtype if outputs else gradient.dtype
    block = AMDStorage(route["capacity"] * width, dtype)
    starts = _host_offsets(route)
    item = 2 if dtype == "bfloat16" else 4
    for expert, values in outputs:
        if values.size:
            block.runtime.copy(block.ptr + starts[expert] * width * item, values.ptr, values.nbytes)
    d_block, d_weights = combine_backward_all(_as_dtype(gradient, dtype), block, route, width)
    grads = []
    for expert, values in outputs:
        part = AMDStorage(values.size, dtype)
        if values.size:
            part.runtime.copy(part.ptr, d_block.ptr + starts[expert] * width * item, values.nbytes)
        grads.append(part)
    return (*grads, d_weights)


def route_gather_backward_all(d_rows, route, width, *, out_dtype=None):
    """Token-row gradient of route_gather_all: the sum over each token's
    slots of its expert-major rows (fp32 sum, one rounding to out_dtype:
    the rows' dtype, or bf16 from fp32 rows)."""
    out_dtype = d_rows.dtype if out_dtype is None else out_dtype
    out = AMDStorage(route["rows"] * width, out_dtype)
    if out.size:
        out.runtime.call("qutai_amd_combine", d_rows.ptr, None, route["indices"].ptr, route["locations"].ptr,
                         route["offsets"].ptr, out.ptr, route["rows"], width, route["top_k"], code(d_rows.dtype),
                         code(out_dtype))
    return out


def routing_backward(gradient, route, auxiliary=False):
    """Gradient of the router logits (cuda_lm.routing_backward,
    cuda_lm.py:452-467): from the routing weights' gradient [rows*top_k], or
    with ``auxiliary`` from the aux loss's scalar gradient."""
    rows, experts = route["rows"], route["experts"]
    g = _as_dtype(gradient, "float32")
    if g.size != (1 if auxiliary else rows * route["top_k"]):
        raise ValueError("routing_backward: gradient size does not match the route")
    out = AMDStorage(rows * experts, "float32")
    if rows:
        out.runtime.call("qutai_amd_route_backward", g.ptr, route["probs"].ptr, route["weights"].ptr,
                         route["indices"].ptr, route["utilization"].ptr, out.ptr, rows, experts, route["top_k"],
                         int(bool(auxiliary)))
    return out


def moe_experts_backward(gradient, route, saved, width, hidden, *, x_dtype, weight_dtype):
    """Backward of moe_experts_forward: (dx, d routing weights, dW_gate,
    dW_up, dW_down).  Every product is one grouped launch over all experts
    (NN for the data gradients, grouped-K TN for the weight gradients); the
    token gradient sums each token's slots in fp32 and rounds once.  Padded
    widths as in the forward; weight gradients are cropped back."""
    wp, hp = _pad8(width), _pad8(hidden)
    experts, capacity = route["experts"], route["capacity"]
    dt = saved["down"].dtype
    d_down, d_weights = combine_backward_all(_as_dtype(gradient, dt), saved["down"], route, width)
    if wp != width:
        d_down = repitch(d_down, 1, capacity, width, capacity, wp)
    d_act = grouped_gemm(d_down, saved["w_down"], route, wp, hp, out_dtype=dt, transpose_right=False)
    dw_down = grouped_gemm_k(d_down, saved["act"], route, wp, hp, out_dtype=weight_dtype)
    d_gate, d_up = silu_mul_backward(d_act, saved["gate"], saved["up"])
    if hp % 64 == 0:  # dGate W_gate + dUp W_up in one accumulator
        d_rows = grouped_gemm_pair(d_gate, d_up, saved["w_gate"], saved["w_up"], route, hp, wp)
    else:
        d_rows = grouped_gemm(d_gate, saved["w_gate"], route, hp, wp, out_dtype="float32", transpose_right=False)
        grouped_gemm(d_up, saved["w_up"], route, hp, wp, out_dtype="float32", transpose_right=False, out=d_rows,
                     accumulate=True)
    gathered = saved.get("gathered", False)
    dw_gate = grouped_gemm_k(d_gate, saved["rows"], route, hp, wp, out_dtype=weight_dtype, gather=gathered)
    dw_up = grouped_gemm_k(d_up, saved["rows"], route, hp, wp, out_dtype=weight_dtype, gather=gathered)
    if (wp, hp) != (width, hidden):
        d_rows = repitch(d_rows, 1, capacity, wp, capacity, width)
        dw_gate, dw_up = (repitch(w, experts, hp, wp, hidden, width) for w in (dw_gate, dw_up))
        dw_down = repitch(dw_down, experts, wp, hp, width, hidden)
    if x_dtype == "bfloat16":  # fp32 slot sums rounded once, straight to bf16
        dx = route_gather_backward_all(d_rows, route, width, out_dtype="bfloat16")
    else:
        dx = _as_dtype(route_gather_backward_all(d_rows, route, width), x_dtype)
    return dx, d_weights, dw_gate, dw_up, dw_down


def _check_attention(q, k, v, batch, time, heads, kv_heads, dim):
    if len({q.dtype, k.dtype, v.dtype}) != 1 or q.dtype not in ("bfloat16", "float32"):
        raise ValueError("attention takes q, k, v of one dtype, bfloat16 or float32")
    if not 0 < dim <= 256 or kv_heads <= 0 or heads % kv_heads:
        raise ValueError("attention needs 0 < head dimension <= 256 and heads divisible by kv_heads")
    if q.size != batch * time * heads * dim or k.size != batch * time * kv_heads * dim or v.size != k.size:
        raise ValueError("q/k/v sizes do not match (batch, time, heads, dim)")


def _on_matrix_cores(dtype, dim):
    """Whether attention of this type and head dimension runs on the matrix
    cores, for the launch counter (sequences of a few positions aside)."""
    return dim % 8 == 0 if dtype == "bfloat16" else dim % 4 == 0 and dim <= 128


def attention(q, k, v, batch, time, heads, kv_heads, dim, *, causal=True, layout=1, scale=None):
    """Attention forward (cuda_lm.attention, src/qutai/backends/cuda_lm.py:229-275):
    (out, lse float32).  bf16 q/k/v with head dimension 64 run the fused MFMA
    kernel; other head dimensions (<= 256) and float32 storage run the MFMA
    kernels that keep fp32 values in bf16 parts; rows that are not 16-byte
    aligned, fp32 above 128 and sequences of a few positions the
    one-wave-per-row kernel, the reference's own fallback shape.
    layout 1 is the lm layout [batch][time][heads][dim], layout 0 the nn
    layout [batch][heads][time][dim].  The score matrix is never stored."""
    _check_attention(q, k, v, batch, time, heads, kv_heads, dim)
    out = AMDStorage(q.size, q.dtype)
    lse = AMDStorage(batch * heads * time, "float32")
    scale = dim ** -0.5 if scale is None else scale
    if q.size:
        out.runtime.call("qutai_amd_attention_fwd", q.ptr, k.ptr, v.ptr, out.ptr, lse.ptr, batch, heads, kv_heads,
                         time, dim, code(q.dtype), layout, float(scale), int(bool(causal)),
                         mfma=_on_matrix_cores(q.dtype, dim))
    return out, lse


# Where one workgroup per (batch, head, query) beats two products around a mask and a softmax.  The
# cache is read again by each query: 32 batches, 16 heads of 128, 4000 keys, bf16, take 487 us against
# 789 for eight queries, and twice that against 852 for 16.  A workgroup reads 67 GB/s where few are in
# flight: 12000 keys of 128 in bf16 (3 MB) take 92 us against 158, keys of 256 188 against 127.
CACHED_LENGTH, CACHED_KEYS, CACHED_BYTES = 8, 12000, 12000 * 128 * 2


def attention_cached_serves(q, k, v, length, total, dim):
    """Whether ``attention_cached`` takes operands of these sizes and types."""
    step = {"bfloat16": 8, "float32": 4}.get(q.dtype)  # elements of 16 bytes
    return (step is not None and q.dtype == k.dtype == v.dtype and 0 < dim <= 256 and dim % step == 0
            and 0 < length <= CACHED_LENGTH and total <= CACHED_KEYS and total * dim * 16 // step <= CACHED_BYTES
            and q.size // dim < 1 << 22  # a workgroup of 1024 threads each, fewer than 2^32 threads in a launch
            and all(x.ptr % 16 == 0 for x in (q, k, v)))


def attention_cached_gains(q, length, total, dim):
    """Whether ``attention_cached`` is faster than the products for operands that
    it takes: for one query, and for fp32, throughout.  Several bf16 queries, in
    ns for each (batch, head): a workgroup costs 8.6 and 0.03 a key of 64, the
    products 10 + 15 and 0.36, and 100 us more of host time (2000 batches, 8 heads
    of 64, a layer call of 8 queries over 8 keys 1582 us and 891 with the products,
    8 over 135 2246 and 1704, 4 over 35 1046 and 1038, 4 over 131 1456 and 1518)."""
    if length == 1 or q.dtype != "bfloat16":
        return True
    pairs, wide = q.size // (length * dim), dim / 64
    queries, products = length * (8.6 + 0.03 * wide * total), 10 + 15 * wide + 0.36 * wide * total
    return pairs * (queries - products) <= 100_000


def attention_cached(q, k, v, batch, length, total, heads, dim):
    """softmax(Q K^T / sqrt(dim)) V of ``length`` new positions over the
    (batch, heads, total, dim) cache that ends with them; q and the result are
    (batch, length, heads, dim) (the products, mask and softmax of
    src/qutai/nn/layers.py:345-355 in one launch)."""
    if not attention_cached_serves(q, k, v, length, total, dim):
        raise ValueError("cached attention does not take these sizes and types")
    if total < length or q.size != batch * length * heads * dim or k.size != batch * total * heads * dim \
            or v.size != k.size:
        raise ValueError("q/k/v sizes do not match the cache's shape")
    out = AMDStorage(q.size, q.dtype)
    if q.size:
        out.runtime.call("qutai_amd_attention_cached", q.ptr, k.ptr, v.ptr, out.ptr, batch, heads, length, total, dim,
                         code(q.dtype), dim ** -0.5)
    return out


def cache_join(past, new, rows):
    """(keys, values) of earlier positions followed by new ones in each of
    ``rows`` (batch, head) rows, in one launch (src/qutai/nn/cache.py:5-29);
    None where rows are not whole 16-byte chunks of one type."""
    stores = (*past, *new)
    dtype, item = past[0].dtype, amd._item(past[0].dtype)
    if not rows or any(x.dtype != dtype or x.ptr % 16 for x in stores) or past[0].size != past[1].size \
            or new[0].size != new[1].size or any(x.size % rows or x.size // rows * item % 16 for x in stores):
        return None
    past_bytes, new_bytes = past[0].size // rows * item, new[0].size // rows * item
    # the launch holds 2 x rows x (16 KiB segments of a row) workgroups of 256 threads, fewer than 2^32 threads
    if not new_bytes or max(past_bytes, new_bytes) > 1 << 34 or rows * -(-(past_bytes + new_bytes) >> 14) >= 1 << 23:
        return None
    out = tuple(AMDStorage(past[0].size + new[0].size, dtype) for _ in range(2))
    out[0].runtime.call("qutai_amd_cache_join", *(x.ptr for x in (*stores, *out)), rows, past_bytes, new_bytes)
    return out


class QuantizedCache:
    """Device memory of a quantised key and value cache: codes of 8 bits (a
    scale per row) or 4 bits (a scale per 32 channels) for ``capacity``
    positions (rounded up to whole blocks of 32) of each (sequence, kv head),
    laid out by the library (qutai_amd_cache_quantize), and the workspace of the
    attention over it."""

    def __init__(self, batch, kv_heads, dim, capacity, bits):
        if bits not in (8, 4):
            raise ValueError("a quantised cache has codes of 8 or 4 bits")
        if batch <= 0 or not 0 < kv_heads <= 65536 or not 0 < dim <= 256 or not 0 < capacity <= 1 << 30:
            raise ValueError("a quantised cache needs sequences, kv heads, a head width up to 256 and a capacity")
        capacity = (capacity + 31) // 32 * 32
        self.batch, self.kv_heads, self.dim, self.capacity, self.bits = batch, kv_heads, dim, capacity, bits
        pitch = get_runtime().lib.qutai_amd_cache_pitch(dim)
        rows, scales = batch * kv_heads * capacity, 1 if bits == 8 else pitch // 32
        # codes are raw bytes: eight to a word (a row has 16 at least)
        self.key_codes, self.value_codes = (AMDStorage(rows * pitch * bits // 64, "int64") for _ in range(2))
        self.key_scales, self.value_scales = (AMDStorage(rows * scales, "bfloat16") for _ in range(2))
        self.workspace = AMDStorage(0, "float32")


def _cache_positions(cache, *arrays):
    for values in arrays:
        if values is not None and (values.dtype != "int64" or values.size != cache.batch):
            raise ValueError("a cache's positions and counts are one int64 per sequence")


def cache_rows(keys, values, batch, new, kv_heads, dim, *, key_column=0, key_row=None, value_column=0, value_row=None):
    """(key_row, value_row) of new keys and values that ``cache_quantize`` takes
    for a cache of these sizes; ValueError where it does not take them."""
    width = kv_heads * dim
    key_row, value_row = (width if row is None else row for row in (key_row, value_row))
    if new < 0 or keys.dtype != values.dtype or keys.dtype not in ("bfloat16", "float32"):
        raise ValueError("cached keys and values are bfloat16 or float32, of one dtype")
    for x, column, row in ((keys, key_column, key_row), (values, value_column, value_row)):
        if column < 0 or column + width > row or x.size < batch * new * row:
            raise ValueError("keys and values need new positions of kv_heads * dim values for every sequence")
    return key_row, value_row


def cache_quantize(cache, keys, values, new, *, start=0, starts=None, counts=None, key_column=0, key_row=None,
                   value_column=0, value_row=None):
    """Quantise ``new`` positions of every sequence into ``cache`` from position
    start + starts[b] on (``starts``, ``counts``: int64 storages of one value per
    sequence; only the first counts[b] positions are written, and none outside
    the capacity).  keys and values are [batch][new][kv_heads][dim], or columns
    key_column .. (value_column ..) of wider matrices of key_row (value_row)
    elements per position."""
    key_row, value_row = cache_rows(keys, values, cache.batch, new, cache.kv_heads, cache.dim, key_column=key_column,
                                    key_row=key_row, value_column=value_column, value_row=value_row)
    _cache_positions(cache, starts, counts)
    if new:
        item = _TYPES[keys.dtype][1]
        cache.key_codes.runtime.call(
            "qutai_amd_cache_quantize", keys.ptr + key_column * item, values.ptr + value_column * item,
            cache.key_codes.ptr, cache.key_scales.ptr, cache.value_codes.ptr, cache.value_scales.ptr, amd._p(starts),
            amd._p(counts), start, cache.batch, new, cache.kv_heads, cache.dim, cache.capacity, key_row, value_row,
            cache.bits, code(keys.dtype))


def cache_dequantize(cache, length, *, lengths=None, shift=0, dtype="float32"):
    """(keys, values) that the cache holds at its first ``length`` positions,
    [batch][kv_heads][length][dim] in ``dtype``; zeros from position shift +
    lengths[b] on (without ``lengths``: from ``length`` on)."""
    if not 0 <= length <= cache.capacity or dtype not in ("bfloat16", "float32"):
        raise ValueError("a cache is read up to its capacity, as bfloat16 or float32")
    _cache_positions(cache, lengths)
    shift = shift if lengths is not None else length
    out = tuple(AMDStorage(cache.batch * cache.kv_heads * length * cache.dim, dtype) for _ in range(2))
    if length:
        out[0].runtime.call("qutai_amd_cache_dequantize", cache.key_codes.ptr, cache.key_scales.ptr, cache.value_codes.ptr,
                            cache.value_scales.ptr, *(x.ptr for x in out), amd._p(lengths), shift, cache.batch,
                            cache.kv_heads, cache.dim, cache.capacity, length, cache.bits, code(dtype))
    return out


def attention_quantized(cache, q, new, heads, *, start=0, starts=None, counts=None, longest=None, scale=None):
    """Attention of ``new`` positions over a quantised cache that holds them:
    q and the result are [batch][new][heads][dim]; query t of sequence b sees
    the cache up to position start + starts[b] + t.  Rows t >= counts[b] are
    zero.  ``longest`` (the capacity if not given) bounds the positions that any
    sequence sees and sizes the split of the work."""
    if q.dtype not in ("bfloat16", "float32"):
        raise ValueError("attention_quantized takes bfloat16 or float32 queries")
    if new < 0 or heads <= 0 or heads % cache.kv_heads or q.size != cache.batch * new * heads * cache.dim:
        raise ValueError("queries need new positions of heads * dim values, heads a multiple of the cache's")
    _cache_positions(cache, starts, counts)
    longest = cache.capacity if longest is None else longest
    if not 0 <= longest <= cache.capacity:
        raise ValueError("longest lies between 0 and the capacity")
    scale = cache.dim ** -0.5 if scale is None else scale
    out = AMDStorage(q.size, q.dtype)
    if q.size:
        runtime, dtype = out.runtime, code(q.dtype)
        need = runtime.attention_workspace(cache.batch, new, heads, cache.kv_heads, cache.dim, longest, dtype)
        if need > cache.workspace.nbytes:
            cache.workspace = AMDStorage((need + 3) // 4, "float32")
        runtime.call("qutai_amd_attention_quantized", q.ptr, cache.key_codes.ptr, cache.key_scales.ptr,
                     cache.value_codes.ptr, cache.value_scales.ptr, out.ptr, amd._p(starts), amd._p(counts), start,
                     cache.batch, new, heads, cache.kv_heads, cache.dim, cache.capacity, longest, cache.bits,
                     dtype, float(scale), cache.workspace.ptr, cache.workspace.nbytes, mfma=True)
    return out


def attention_backward(gradient, q, k, v, out, lse, batch, time, heads, kv_heads, dim, *, causal=True, layout=1,
                       scale=None):
    """(dq, dk, dv) of ``attention`` (cuda_lm.attention_backward,
    src/qutai/backends/cuda_lm.py:278-365): activations and gradient of one
    dtype, float32 lse from the forward (the reference's ValueError rule,
    cuda_lm.py:279-282); deterministic."""
    _check_attention(q, k, v, batch, time, heads, kv_heads, dim)
    if gradient.dtype != q.dtype or out.dtype != q.dtype or lse.dtype != "float32":
        raise ValueError("attention backward needs gradient/out of the activations' dtype and a float32 lse")
    if gradient.size != q.size or out.size != q.size or lse.size != batch * time * heads:
        raise ValueError("gradient/out/lse sizes do not match (batch, time, heads, dim)")
    dq, dk, dv = AMDStorage(q.size, q.dtype), AMDStorage(k.size, k.dtype), AMDStorage(v.size, v.dtype)
    delta = AMDStorage(lse.size, "float32")
    scale = dim ** -0.5 if scale is None else scale
    if q.size:
        runtime = dq.runtime
        need = runtime.lib.qutai_amd_attention_bwd_workspace_size(batch, heads, kv_heads, time, dim, code(q.dtype))
        workspace = AMDStorage((need + 3) // 4, "float32") if need else None
        runtime.call("qutai_amd_attention_bwd", gradient.ptr, q.ptr, k.ptr, v.ptr, out.ptr, lse.ptr, dq.ptr, dk.ptr,
                     dv.ptr, delta.ptr, workspace.ptr if workspace else None, need, batch, heads, kv_heads, time, dim,
                     code(q.dtype), layout, float(scale), int(bool(causal)), mfma=_on_matrix_cores(q.dtype, dim))
    return dq, dk, dv


def _packed_places(q, k, v, packing, heads, kv_heads, dim, q_column, q_row, k_column, k_row, v_column, v_row):
    """Addresses of the first q, k and v rows of a packed call, which it checks, the
    elements from row to row, and all of them or'd in bytes: whole 16-byte chunks if
    that is."""
    dtype = q.dtype
    if dtype not in ("bfloat16", "float32") or k.dtype != dtype or v.dtype != dtype:
        raise ValueError("attention takes q, k, v of one dtype, bfloat16 or float32")
    if not 0 < dim <= 256 or kv_heads <= 0 or heads <= 0 or heads % kv_heads:
        raise ValueError("attention needs 0 < head dimension <= 256 and heads divisible by kv_heads")
    total = packing.total
    q_at, q_row = _qk_rows(q, total, heads, dim, q_column, q_row, dtype)
    k_at, k_row = _qk_rows(k, total, kv_heads, dim, k_column, k_row, dtype)
    v_at, v_row = _qk_rows(v, total, kv_heads, dim, v_column, v_row, dtype)
    return q_at, k_at, v_at, q_row, k_row, v_row, q_at | k_at | v_at | (q_row | k_row | v_row | dim) * _TYPES[dtype][1]


def _packed_tail(packing, *blocks):
    """Zeros in the rows behind the last sequence of contiguous results."""
    for x in blocks:
        if x is not None:
            width = x.size // packing.total
            start = packing.used * width
            x.runtime.call("qutai_amd_fill", x.ptr + start * _TYPES[x.dtype][1], x.size - start, 0.0, code(x.dtype))


def attention_packed(q, k, v, packing, heads, kv_heads, dim, *, causal=True, scale=None, q_column=0, q_row=None,
                     k_column=0, k_row=None, v_column=0, v_row=None, rest=False):
    """(out, lse float32) of attention among the tokens of each sequence of a
    ``packing`` (an ``lm.Packing``): as ``attention``, with the sequences one
    behind the other in the rows of q, k and v, which may be columns q_column ..
    of matrices of q_row elements per token (and so on).  out is contiguous
    [total][heads][dim], lse [total][heads]; rows behind the last sequence are
    zero.  With ``rest`` also what out's rounding left, for the backward (None
    where there is none).  bf16 heads of up to 128 channels round probabilities (and
    dS) to bf16 for their products, in two parts in sequences of up to 64 tokens."""
    q_at, k_at, v_at, q_row, k_row, v_row, odd = _packed_places(q, k, v, packing, heads, kv_heads, dim, q_column, q_row,
                                                                k_column, k_row, v_column, v_row)
    name, total = q.dtype, packing.total
    out, lse, left, dtype = AMDStorage(total * heads * dim, name), AMDStorage(total * heads, "float32"), None, code(name)
    scale = dim ** -0.5 if scale is None else float(scale)
    if packing.used:
        tiles, count, rows, _ = packing.plan(0, heads, kv_heads, dim, dtype, odd % 16 == 0, scale, causal)
        if rest and rows > 4 and name == "bfloat16" and dim <= 128:
            left = AMDStorage(out.size, name)
        out.runtime.call("qutai_amd_attention_packed_fwd", q_at, k_at, v_at, out.ptr, lse.ptr, amd._p(left), tiles.ptr, count,
                         rows, *packing.extent, heads, kv_heads, dim, q_row, k_row, v_row, dtype, scale, int(bool(causal)),
                         mfma=rows > 4)
    if packing.used < total:
        _packed_tail(packing, out, lse, left)
    return (out, lse, left) if rest else (out, lse)


def attention_packed_backward(gradient, q, k, v, out, lse, packing, heads, kv_heads, dim, *, causal=True, scale=None,
                              q_column=0, q_row=None, k_column=0, k_row=None, v_column=0, v_row=None, rest=None,
                              into=None):
    """(dq, dk, dv) of ``attention_packed``: its operands and options, its out, lse
    and rest, and the contiguous gradient of out.  The results are contiguous, or
    with ``into`` (a storage laid out as the one matrix that q, k and v are columns
    of) its columns q_column .., k_column .., v_column ...; every one is summed in
    a fixed order.  Rows behind the last sequence are zero."""
    columns = q_column, k_column, v_column
    q_at, k_at, v_at, q_row, k_row, v_row, odd = _packed_places(q, k, v, packing, heads, kv_heads, dim, q_column, q_row,
                                                                k_column, k_row, v_column, v_row)
    total, widths = packing.total, (heads * dim, kv_heads * dim, kv_heads * dim)
    if gradient.dtype != q.dtype or out.dtype != q.dtype or lse.dtype != "float32":
        raise ValueError("attention backward needs gradient/out of the activations' dtype and a float32 lse")
    if gradient.size != total * heads * dim or out.size != gradient.size or lse.size != total * heads:
        raise ValueError("gradient/out/lse sizes do not match (total, heads, dim)")
    if rest is not None and (rest.dtype != q.dtype or rest.size != out.size):
        raise ValueError("rest is what attention_packed returned beside out")
    if into is None:
        results = tuple(AMDStorage(total * width, q.dtype) for width in widths)
        targets, steps = tuple(x.ptr for x in results), widths
    else:
        spans = sorted((column, column + width) for column, width in zip(columns, widths))
        if not q_row == k_row == v_row or any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("into holds the gradients in separate columns of one row")
        for x in (gradient, q, k, v, out, *(() if rest is None else (rest,))):
            if into.ptr < x.ptr + x.nbytes and x.ptr < into.ptr + into.nbytes:
                raise ValueError("into must not share memory with an input")
        results, steps = (into,) * 3, (q_row,) * 3
        targets = tuple(_qk_rows(into, total, n, dim, column, q_row, q.dtype)[0]
                        for column, n in zip(columns, (heads, kv_heads, kv_heads)))
    for at in (*targets, gradient.ptr, out.ptr):
        odd |= at
    dtype = code(q.dtype)
    scale = dim ** -0.5 if scale is None else float(scale)
    if packing.used:
        delta = AMDStorage(total * heads, "float32")
        (q_tiles, q_count, q_rows, _), (k_tiles, k_count, k_rows, need) = (
            packing.plan(n, heads, kv_heads, dim, dtype, odd % 16 == 0, scale, causal) for n in (1, 2))
        workspace = AMDStorage(need // 4, "float32") if need else None
        if rest is not None and rest.ptr % 16 and odd % 16 == 0:  # read with the others' whole chunks
            rest = copy_rows(rest, 1, rest.size)
        delta.runtime.call("qutai_amd_attention_packed_bwd", gradient.ptr, q_at, k_at, v_at, out.ptr, amd._p(rest), lse.ptr,
                           *targets, delta.ptr, amd._p(workspace), need, q_tiles.ptr, q_count, q_rows, k_tiles.ptr, k_count,
                           k_rows, *packing.extent, heads, kv_heads, dim, q_row, k_row, v_row, *steps, dtype, scale, int(bool(causal)),
                           mfma=max(q_rows, k_rows) > 4)
    if packing.used < total:
        if into is None:
            _packed_tail(packing, *results)
        else:
            for at, width in zip(targets, widths):
                _zero_columns(into, at, total - packing.used, packing.used, q_row, width)
    return results


def _zero_columns(block, at, rows, first, row, width):
    """Zeros in ``rows`` rows from ``first`` on of the columns that start at
    address ``at`` of a matrix of ``row`` elements per row."""
    zeros = amd.full(rows * width, 0.0, dtype=block.dtype)
    column = (at - block.ptr) // _TYPES[block.dtype][1]
    amd._copy_strided(zeros, block, (rows, width), (width, 1), (row, 1), source_offset=0, target_offset=first * row + column)


# ---- decoder glue (the rest of a Decoder.loss step) ---------------------------------

def _acc_dtype(dtype):
    """Accumulation dtype of the activations (cuda_lm.py:9-11): fp32 for bf16/fp32."""
    if dtype not in ("bfloat16", "float32"):
        raise ValueError("amd lm kernels take bfloat16 or float32 activations")
    return "float32"


def add_into(target, source):
    """target += source, element-wise in target's dtype (cuda_lm.py:64-73)."""
    if target.dtype != source.dtype or target.size != source.size:
        raise ValueError("add_into needs storages of equal dtype and size")
    if target.size:
        target.runtime.call("qutai_amd_add", target.ptr, source.ptr, target.ptr, target.size, code(target.dtype))


def embedding(weight, ids, width, *, out_dtype=None):
    """Rows of the fp32 embedding table for the host token ids
    (cuda_lm.py:77-93), in out_dtype (default the table's)."""
    dtype = out_dtype or weight.dtype
    if _acc_dtype(dtype) != weight.dtype:
        raise ValueError("the embedding table must be in the activations' accumulation dtype")
    if not (isinstance(ids, array) and ids.typecode == "q"):
        ids = array("q", (int(t) for t in ids))
    result = AMDStorage(len(ids) * width, dtype)
    if result.size:
        identifiers = amd.storage(ids, dtype="int64")
        result.runtime.call("qutai_amd_embedding", weight.ptr, identifiers.ptr, result.ptr, len(ids), width,
                            code(dtype))
    return result


def embedding_backward_index(ids):
    """Device index of the table gradient's row sums: the distinct token ids
    ascending, offsets into the rows, and the rows of each token in input
    order (cuda_lm.py:96-123 groups them the same way on the host).  Built
    with C-level sorts and searches; made once per forward, so the backward
    launches without a host transfer."""
    if not (isinstance(ids, array) and ids.typecode == "q"):
        ids = array("q", (int(t) for t in ids))
    order = sorted(range(len(ids)), key=ids.__getitem__)  # stable: input order within a token
    grouped = array("q", map(ids.__getitem__, order))
    # a token's rows start where the grouped ids change
    offsets = array("q", range(min(1, len(ids))))
    offsets.extend(compress(range(1, len(ids)), map(ne, islice(grouped, 1, None), grouped)))
    tokens = array("q", map(grouped.__getitem__, offsets))
    offsets.append(len(ids))
    return tuple(amd.storage(values, dtype="int64") for values in (tokens, offsets, array("q", order)))


def embedding_backward(gradient, ids, count, width, *, index=None, out=None):
    """Table gradient [count][width] (fp32): each token's gradient rows summed
    in input order (cuda_lm.py:96-123).  ``index`` is
    ``embedding_backward_index(ids)`` when the caller made it earlier; with
    ``out`` (an fp32 [count][width] storage) the row sums are added into it in
    place and it is returned."""
    if out is None:
        result = amd.full(count * width, 0.0, dtype=_acc_dtype(gradient.dtype))
    elif out.dtype != "float32" or out.size != count * width:
        raise ValueError("embedding_backward accumulates into an fp32 [count][width] storage")
    else:
        result = out
    if len(ids) and width:
        tokens, offsets, positions = embedding_backward_index(ids) if index is None else index
        result.runtime.call("qutai_amd_embedding_backward", gradient.ptr, tokens.ptr, offsets.ptr, positions.ptr,
                            result.ptr, tokens.size, width, code(gradient.dtype), int(out is not None))
    return result


class EmbeddingRowSums(DeferredGradient):
    """The table gradient of an embedding lookup as a deferred contribution:
    dense on demand, or its rows added in place into a gradient the backward
    pass has just made (a tied embedding/head table), which skips filling a
    [count][width] zero buffer and adding two whole tables."""

    device = "amd"
    dtype = "float32"

    def __init__(self, gradient, ids, count, width, index):
        self.gradient, self.ids, self.count, self.width, self.index = gradient, ids, count, width, index
        self.size = count * width

    def materialize(self):
        return embedding_backward(self.gradient, self.ids, self.count, self.width, index=self.index)

    def add_into(self, storage):
        embedding_backward(self.gradient, self.ids, self.count, self.width, index=self.index, out=storage)


def rms_norm(values, weight, width, eps, *, bf16_copy=False):
    """(out, inverse) of RMSNorm over rows of width (cuda_lm.py:126-145); both
    fp32.  With ``bf16_copy`` also out rounded to bf16 (the copy the bf16
    path's products take), written by the same kernel: (out, inverse, copy)."""
    acc = _acc_dtype(values.dtype)
    if weight.dtype != acc or weight.size != width:
        raise ValueError("rms_norm needs an fp32 weight of width values")
    rows = values.size // width
    out, inverse = AMDStorage(values.size, acc), AMDStorage(rows, acc)
    copy = AMDStorage(values.size, "bfloat16") if bf16_copy else None
    if rows:
        out.runtime.call("qutai_amd_rms_norm_bf16", values.ptr, weight.ptr, out.ptr, None if copy is None else copy.ptr,
                         inverse.ptr, rows, width, float(eps), code(values.dtype))
    return (out, inverse, copy) if bf16_copy else (out, inverse)


def rms_norm_backward(gradient, values, weight, inverse, width, residual=None):
    """(dx in the activation dtype, dweight fp32) (cuda_lm.py:148-177).  With
    ``residual`` (fp32 activations only) dx is residual + dx, added as dx is
    stored: one fp32 rounding, the value of a separate add."""
    rows = values.size // width
    g = gradient if gradient.dtype == "float32" else amd.from_storage(gradient, dtype="float32")
    if residual is not None and (values.dtype != "float32" or residual.dtype != "float32"
                                 or residual.size != values.size):
        raise ValueError("the residual gradient must be fp32 of the activation's size")
    dx, dw = AMDStorage(values.size, values.dtype), AMDStorage(width, weight.dtype)
    if rows:
        runtime = get_runtime()
        partial = AMDStorage(runtime.lib.qutai_amd_rms_norm_workspace(rows, width), "float32")
        runtime.call("qutai_amd_rms_norm_backward", g.ptr, values.ptr, weight.ptr, inverse.ptr,
                     None if residual is None else residual.ptr, dx.ptr, dw.ptr, partial.ptr, rows, width,
                     code(values.dtype))
    elif residual is not None:
        dx = residual.copy()
    return dx, dw


def silu(values):
    """x * sigmoid(x) (cuda_lm.py:180-192)."""
    out = AMDStorage(values.size, values.dtype)
    if values.size:
        out.runtime.call("qutai_amd_silu", values.ptr, None, out.ptr, values.size, 0, code(values.dtype))
    return out


def silu_backward(gradient, values):
    """g * s * (1 + x (1 - s)) (cuda_lm.py:195-207)."""
    out = AMDStorage(values.size, values.dtype)
    if values.size:
        out.runtime.call("qutai_amd_silu", values.ptr, gradient.ptr, out.ptr, values.size, 1, code(values.dtype))
    return out


def rope(values, batch, time, heads, dim, theta, offset=0, inverse=False, *, column=0, row=None, out=None,
         out_column=0, out_row=None):
    """Rotary embedding of [batch][time][heads][dim] (cuda_lm.py:210-226).
    ``values`` may be a wider matrix of ``row`` elements per position whose
    columns column .. column + heads*dim are rotated; the result goes to a new
    contiguous block, or into columns out_column .. of ``out`` (``out_row``
    elements per position)."""
    width = heads * dim
    row = width if row is None else row
    positions = batch * time
    if column < 0 or row < width or column + width > row or values.size < positions * row:
        raise ValueError("rope columns outside the source rows")
    if out is None:
        if out_column or out_row not in (None, width):
            raise ValueError("a new rope result is contiguous")
        out, out_row = AMDStorage(positions * width, values.dtype), width
    else:
        out_row = width if out_row is None else out_row
        if out.dtype != values.dtype or out_column < 0 or out_row < width or out_column + width > out_row \
                or out.size < positions * out_row:
            raise ValueError("rope output columns outside the target rows")
    if positions * width:
        item = _TYPES[values.dtype][1]
        out.runtime.call("qutai_amd_rope_rows", values.ptr + column * item, out.ptr + out_column * item, batch, time,
                         heads, dim, float(theta), offset, int(bool(inverse)), row, out_row, code(values.dtype))
    return out


def _qk_rows(values, positions, heads, dim, column, row, dtype):
    """(pointer, elements per position) of one side's head rows: columns
    column .. column + heads*dim of ``values``; (None, 0) without heads."""
    if not heads:
        return None, 0
    width = heads * dim
    row = width if row is None else row
    if values.dtype != dtype or column < 0 or column + width > row or values.size < positions * row:
        raise ValueError("query and key rows need one dtype and columns inside their storages")
    return values.ptr + column * _TYPES[dtype][1], row


def _qk_arguments(q, k, q_weight, k_weight, batch, time, heads, kv_heads, dim, starts):
    sides = [(x, w) for x, w, n in ((q, q_weight, heads), (k, k_weight, kv_heads)) if n]
    if min(batch, time, heads, kv_heads) < 0 or not sides or dim <= 0 or dim % 2 or dim > 256:
        raise ValueError("qk_norm_rope needs query or key heads of an even width up to 256")
    dtype = sides[0][0].dtype
    if dtype not in ("bfloat16", "float32"):
        raise ValueError("qk_norm_rope takes bfloat16 or float32 rows")
    weights = [w for _, w in sides if w is not None]
    if len(weights) not in (0, len(sides)) or any(w.dtype != "float32" or w.size != dim for w in weights):
        raise ValueError("qk_norm_rope takes fp32 weights of dim values for every side, or none")
    if starts is not None and (starts.dtype != "int64" or starts.size != batch):
        raise ValueError("starts holds one int64 position per sequence")
    return dtype


def qk_norm_rope(q, k, q_weight, k_weight, batch, time, heads, kv_heads, dim, theta, eps=1e-6, *, offset=0, starts=None,
                 q_column=0, q_row=None, k_column=0, k_row=None):
    """RMSNorm of every query and key head (rows of ``dim``, an fp32 weight of
    ``dim`` values for each side) and its rotary embedding, one launch and one
    rounding: (q, k), contiguous [batch][time][heads][dim].  Position t of
    sequence b is offset + t, plus ``starts[b]`` (int64 storage) where given.  q
    and k may be columns q_column .. (k_column ..) of a wider matrix of q_row
    (k_row) elements per position, as in ``rope``.  Weights of None leave the
    norm out; 0 heads leave a side out (its result is None)."""
    dtype = _qk_arguments(q, k, q_weight, k_weight, batch, time, heads, kv_heads, dim, starts)
    positions = batch * time
    (q_at, q_row), (k_at, k_row) = (_qk_rows(q, positions, heads, dim, q_column, q_row, dtype),
                                    _qk_rows(k, positions, kv_heads, dim, k_column, k_row, dtype))
    out_q, out_k = (AMDStorage(positions * n * dim, dtype) if n else None for n in (heads, kv_heads))
    if positions:
        get_runtime().call("qutai_amd_qk_norm_rope", q_at, k_at, amd._p(q_weight), amd._p(k_weight), amd._p(out_q),
                           amd._p(out_k), amd._p(starts), offset, batch, time, heads, kv_heads, dim, q_row, k_row,
                           float(theta), float(eps), code(dtype))
    return out_q, out_k


def qk_norm_rope_backward(gq, gk, q, k, q_weight, k_weight, batch, time, heads, kv_heads, dim, theta, eps=1e-6, *,
                          offset=0, starts=None, q_column=0, q_row=None, k_column=0, k_row=None, out=None):
    """(dq, dk, dq_weight, dk_weight) of ``qk_norm_rope``: gq and gk the
    contiguous gradients of its results in the rows' dtype, the other arguments
    its own.  The input gradients are new contiguous storages, or with ``out`` (a
    storage laid out like the wider matrix that holds both q and k: q_row and
    k_row elements per position) its columns q_column .. and k_column ..; the
    weights' gradients (None without weights) are fp32 sums over all rows in a
    fixed order."""
    dtype = _qk_arguments(q, k, q_weight, k_weight, batch, time, heads, kv_heads, dim, starts)
    positions = batch * time
    for g, n in ((gq, heads), (gk, kv_heads)):
        if n and (g.dtype != dtype or g.size != positions * n * dim):
            raise ValueError("gq and gk need the rows' dtype and one value for each of theirs")
    (q_at, q_step), (k_at, k_step) = (_qk_rows(q, positions, heads, dim, q_column, q_row, dtype),
                                      _qk_rows(k, positions, kv_heads, dim, k_column, k_row, dtype))
    if out is None:
        dq, dk = (AMDStorage(positions * n * dim, dtype) if n else None for n in (heads, kv_heads))
        (dq_at, dq_step), (dk_at, dk_step) = (amd._p(dq), heads * dim), (amd._p(dk), kv_heads * dim)
    else:
        if heads and kv_heads and (q_step != k_step or not (q_column + heads * dim <= k_column
                                                            or k_column + kv_heads * dim <= q_column)):
            raise ValueError("out holds q's and k's gradients in separate columns of one row")
        for x in (gq, gk, q, k):
            if x is not None and out.nbytes and out.ptr < x.ptr + x.nbytes and x.ptr < out.ptr + out.nbytes:
                raise ValueError("out must not share memory with an input")
        dq = out if heads else None
        dk = out if kv_heads else None
        (dq_at, dq_step), (dk_at, dk_step) = (_qk_rows(out, positions, heads, dim, q_column, q_row, dtype),
                                              _qk_rows(out, positions, kv_heads, dim, k_column, k_row, dtype))
    dwq, dwk = (AMDStorage(dim, "float32") if n and w is not None else None
                for n, w in ((heads, q_weight), (kv_heads, k_weight)))
    runtime = get_runtime()
    need = runtime.lib.qutai_amd_qk_norm_rope_workspace(dim) if dwq is not None or dwk is not None else 0
    workspace = AMDStorage(need, "float32") if need else None
    runtime.call("qutai_amd_qk_norm_rope_backward", amd._p(gq), amd._p(gk), q_at, k_at, amd._p(q_weight),
                 amd._p(k_weight), dq_at, dk_at, amd._p(dwq), amd._p(dwk), amd._p(starts), offset, batch, time, heads,
                 kv_heads, dim, q_step, k_step, dq_step, dk_step, float(theta), float(eps), code(dtype),
                 amd._p(workspace), need)
    return dq, dk, dwq, dwk


def _int64(value):
    """A whole number as the int that an int64 argument holds."""
    try:
        whole = int(value)
    except (TypeError, ValueError, OverflowError):
        whole = None
    if whole is None or whole != value or not -(1 << 63) <= whole < 1 << 63:
        raise ValueError("the offset is an integer of 64 bits")
    return whole


def rotary(q, k, rotary, batch, time, heads, kv_heads, dim, *, positions=None, offset=0, starts=None, inverse=False,
           q_column=0, q_row=None, k_column=0, k_row=None, out=None, out_row=None, out_q_column=0, out_k_column=None):
    """(q, k) with the first channels of every head turned by their tokens'
    positions as ``rotary`` (an ``lm.Rotary``) says, in one launch; ``inverse``
    turns back, which is the gradient.  Token t of sequence b is at positions[b *
    time + t] (int64 storage of one per token), or at offset + t plus starts[b]
    (int64 storage of one per sequence).  q and k are columns q_column .. and
    k_column .. of matrices of q_row (k_row) elements per token.  The results are
    contiguous [batch][time][heads][dim], or with ``out`` its columns out_q_column
    .. and out_k_column .. (out_row elements per token; ``out`` may be the matrix
    that q and k are columns of, if they are the same columns).  0 heads leave a
    side out (its result is None)."""
    if rotary.dim != dim or min(batch, time, heads, kv_heads) < 0 or heads + kv_heads == 0:
        raise ValueError("rotary turns query or key heads of its own width")
    if inverse not in (False, True):
        raise ValueError("inverse is True or False")
    offset = _int64(offset)
    tokens = batch * time
    if positions is not None and (starts is not None or offset or positions.dtype != "int64" or positions.size != tokens):
        raise ValueError("positions hold one int64 for every token, without offset and starts")
    if starts is not None and (starts.dtype != "int64" or starts.size != batch):
        raise ValueError("starts holds one int64 position per sequence")
    dtype = (q if heads else k).dtype
    if dtype not in ("bfloat16", "float32"):
        raise ValueError("rotary takes bfloat16 or float32 rows")
    q_at, q_step = _qk_rows(q, tokens, heads, dim, q_column, q_row, dtype)
    k_at, k_step = _qk_rows(k, tokens, kv_heads, dim, k_column, k_row, dtype)
    if out is None:
        q_out, k_out = heads * dim, kv_heads * dim
        results = (AMDStorage(tokens * q_out, dtype) if heads else None, AMDStorage(tokens * k_out, dtype) if kv_heads else None)
        q_to, k_to = amd._p(results[0]), amd._p(results[1])
    else:
        q_to, q_out = _qk_rows(out, tokens, heads, dim, out_q_column, out_row, dtype)
        k_to, k_out = _qk_rows(out, tokens, kv_heads, dim, heads * dim if out_k_column is None else out_k_column, out_row, dtype)
        for x, n, source, target in ((q, heads, (q_at, q_step), (q_to, q_out)), (k, kv_heads, (k_at, k_step), (k_to, k_out))):
            if n and source != target and out.ptr < x.ptr + x.nbytes and x.ptr < out.ptr + out.nbytes:
                raise ValueError("out shares memory with an input that is not in its place")
        item = _TYPES[dtype][1]
        if heads and kv_heads and (q_out != k_out or not (q_to + heads * dim * item <= k_to
                                                          or k_to + kv_heads * dim * item <= q_to)):
            raise ValueError("out holds q's and k's results in separate columns of one row")
        results = out if heads else None, out if kv_heads else None
    if tokens:
        get_runtime().call("qutai_amd_rotary", q_at, k_at, q_to, k_to, rotary.turns, amd._p(positions), amd._p(starts),
                           offset, batch, time, heads, kv_heads, dim, rotary.rotary_dim, q_step, k_step, q_out, k_out,
                           int(rotary.layout == "half"), rotary.magnitude, int(inverse), code(dtype))
    return results


class AdamWMoments:
    """Device memory of one tensor's moments: fp32, or 8-bit codes and an exponent
    for every 256 values of each, laid out by the library."""

    def __init__(self, size, bits):
        self.size, self.bits = size, bits
        if bits == 32:
            self.first, self.second = (amd.full(size, 0.0, dtype="float32") for _ in range(2))
            self.exponents = None
        else:  # bytes, as whole int64 words of zeros
            self.first, self.second = (amd.full((size + 7) // 8, 0, dtype="int64") for _ in range(2))
            self.exponents = amd.full((2 * ((size + 255) // 256) + 7) // 8, 0, dtype="int64")
        self.pointers = self.first.ptr, self.second.ptr, amd._p(self.exponents)

    def storages(self):
        return (self.first, self.second) if self.exponents is None else (self.first, self.second, self.exponents)

    def values(self):
        """(first, second) as fp32 storages."""
        if self.bits == 32:
            return self.first, self.second
        out = AMDStorage(self.size, "float32"), AMDStorage(self.size, "float32")
        if self.size:
            out[0].runtime.call("qutai_amd_adamw_moments", self.first.ptr, self.second.ptr, self.exponents.ptr,
                                out[0].ptr, out[1].ptr, self.size)
        return out


def adamw_workspace(count, values):
    """What ``adamw`` needs to cut the norm of up to ``count`` gradients of
    ``values`` values: (partial sums, the norm), fp64 storages."""
    return AMDStorage(get_runtime().lib.qutai_amd_adamw_workspace(count, values), "float64"), amd.full(1, 0.0, dtype="float64")


def adamw(tensors, bits, lr, beta1, beta2, eps, weight_decay, step, *, seed=0, max_norm=None, workspace=None):
    """One AdamW step (its ``step``-th, from 1) over ``tensors``: tuples of a
    parameter's storage, its gradient's, its AdamWMoments and the number that
    tells it from the others where 8-bit codes are rounded.  Parameters and moments
    are changed in place.  With ``max_norm`` returns the fp64 storage that holds the
    norm of all gradients, else None; ``workspace``: an ``adamw_workspace`` of as
    many tensors and values at least, which this step alone uses meanwhile."""
    rows, values = [], 0
    for p, g, moments, index in tensors:
        dtype, size = p.dtype, p._size
        if dtype not in _ADAMW_CODES or g.dtype != dtype or not size == g._size == moments.size or moments.bits != bits:
            raise ValueError("adamw takes float32 or bfloat16 parameters with gradients and moments of their size")
        rows += (p.ptr, g.ptr, *moments.pointers, size, _ADAMW_CODES[dtype], index)
        values += size
    table, partial, norm = array("q", rows), None, None
    if max_norm is not None:
        partial, norm = adamw_workspace(len(rows) // 8, values) if workspace is None else workspace
        if not values:
            norm = amd.full(1, 0.0, dtype="float64")
    if values:
        get_runtime().call("qutai_amd_adamw", table.buffer_info()[0], len(rows) // 8, bits, lr, beta1, beta2, eps,
                           weight_decay, step, seed, max_norm or 0.0, None if partial is None else partial.ptr,
                           0 if partial is None else partial.size, None if norm is None else norm.ptr)
    return norm


_ADAMW_CODES = {name: code(name) for name in ("float32", "bfloat16")}


def copy_rows(source, rows, width, *, column=0, row=None, out=None, out_column=0, out_row=None):
    """Columns column .. column + width of the ``rows`` rows of ``source``
    (``row`` elements each) into a new contiguous [rows][width] block, or into
    columns out_column .. of ``out`` (``out_row`` elements per row)."""
    row = width if row is None else row
    if column < 0 or row < width or column + width > row or source.size < rows * row:
        raise ValueError("copied columns outside the source rows")
    if out is None:
        out, out_column, out_row = AMDStorage(rows * width, source.dtype), 0, width
    else:
        out_row = width if out_row is None else out_row
        if out.dtype != source.dtype or out_column < 0 or out_column + width > out_row or out.size < rows * out_row:
            raise ValueError("copied columns outside the target rows")
    amd._copy_strided(source, out, (rows, width), (row, 1), (out_row, 1), source_offset=column,
                      target_offset=out_column)
    return out


def head_rows(values, start, count, width, time):
    """Rows start .. start+count of the prediction positions (cuda_lm.py:584-598)."""
    result = AMDStorage(count * width, values.dtype)
    if result.size:
        result.runtime.call("qutai_amd_head_rows", values.ptr, result.ptr, count, start, width, time, 0,
                            code(values.dtype))
    return result


def head_rows_backward(target, gradient, start, count, width, time):
    """target[prediction rows] += gradient (cuda_lm.py:601-613)."""
    if count * width:
        target.runtime.call("qutai_amd_head_rows", gradient.ptr, target.ptr, count, start, width, time, 1,
                            code(target.dtype))


def prepare_labels(labels):
    """Labels resident on the device as int64 (cuda_lm.py:616-617)."""
    if not (isinstance(labels, array) and labels.typecode == "q"):
        labels = array("q", (int(x) for x in labels))
    return amd.storage(labels, dtype="int64")


def _head_labels(labels, start, rows):
    ids = labels if isinstance(labels, AMDStorage) else prepare_labels(labels)
    if ids.dtype != "int64" or start < 0 or start + rows > ids.size:
        raise ValueError("invalid head label storage or range")
    return ids, ids.ptr + 8 * start


def head_loss(logits, labels, rows, vocab, *, start=0):
    """Summed cross entropy of rows of logits (label -100 ignored), one fp32
    value (cuda_lm.py:629-643)."""
    _, pointer = _head_labels(labels, start, rows)
    values = AMDStorage(rows, _acc_dtype(logits.dtype))
    if rows:
        values.runtime.call("qutai_amd_head_loss", logits.ptr, pointer, values.ptr, rows, vocab, code(logits.dtype))
    return amd.sum_all(values) if rows else amd.full(1, 0.0, dtype=values.dtype)


def head_block_stats(logits, labels, stats, picked, rows, cols, col0, *, first):
    """Fold one vocabulary block [rows][cols] (columns col0 ..) of the logits
    into the per-row running (max, sum exp) pairs ``stats`` ([rows][2] fp32)
    and the label logits ``picked`` ([rows] fp32)."""
    ids, _ = _head_labels(labels, 0, rows)
    if rows:
        logits.runtime.call("qutai_amd_head_block_stats", logits.ptr, ids.ptr, stats.ptr, picked.ptr, rows, cols, col0,
                            int(first), code(logits.dtype))


def head_block_loss(stats, picked, labels, rows):
    """Summed cross entropy of the rows from their folded stats (one fp32 value)."""
    ids, _ = _head_labels(labels, 0, rows)
    values = AMDStorage(rows, "float32")
    if rows:
        values.runtime.call("qutai_amd_head_block_loss", stats.ptr, picked.ptr, ids.ptr, values.ptr, rows)
    return amd.sum_all(values) if rows else amd.full(1, 0.0, dtype="float32")


def head_block_gradient(logits, labels, stats, gradient, rows, cols, col0, count):
    """In place over one vocabulary block: g / count * (softmax - onehot)."""
    ids, _ = _head_labels(labels, 0, rows)
    g = gradient if gradient.dtype == "float32" else amd.from_storage(gradient, dtype="float32")
    if rows:
        logits.runtime.call("qutai_amd_head_block_gradient", logits.ptr, ids.ptr, stats.ptr, g.ptr, rows, cols, col0,
                            1.0 / count, code(logits.dtype))
    return logits


def _sampling_parameter(value, name, rows, dtype, valid):
    """(device pointer or None, number) of a parameter that is one number or a
    storage of one per row."""
    if isinstance(value, AMDStorage):
        if value.dtype != dtype or value.size != rows:
            raise ValueError(f"{name} for every row is a {dtype} storage of that many values")
        return value.ptr, 0
    if not isinstance(value, (int, float)) or isinstance(value, bool) or not valid(value):
        raise ValueError(f"{name} is out of range")
    return None, value


def sample(logits, uniforms, rows, vocab, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens int64, probabilities float32): one token for each row of
    [rows][vocab] logits, picked by ``uniforms`` (float32 or float64 numbers in
    [0, 1), one per row) among the tokens that are kept.  In the order of falling
    logits (equal ones: lowest index first) ``top_k`` keeps that many (0: all),
    ``top_p`` the shortest prefix of them that holds this share of their weight
    exp((logit - max) / temperature), ``min_p`` those of them that weigh at least
    that much of the largest.  The token is the first, by index, at which the
    running sum of the kept weights exceeds the row's number times their sum; the
    probability is its share.  Temperature 0 takes the largest logit.  Each
    parameter is a number, or a storage of one per row (float32; top_k int64).  A
    NaN logit counts as -inf; a row of -inf gives token -1."""
    if logits.dtype not in ("bfloat16", "float32") or uniforms.dtype not in ("float32", "float64"):
        raise ValueError("sample takes bfloat16 or float32 logits and float32 or float64 uniforms")
    if rows < 0 or not 0 < vocab <= 1 << 20 or rows >= 1 << 22 or logits.size != rows * vocab or uniforms.size != rows:
        raise ValueError("sample needs rows * vocab logits (vocab at most 2^20) and a number for every row")
    temperatures, temperature = _sampling_parameter(temperature, "temperature", rows, "float32",
                                                    lambda x: 0 <= x < float("inf"))
    top_ks, top_k = _sampling_parameter(top_k, "top_k", rows, "int64", lambda x: type(x) is int and 0 <= x < 1 << 62)
    top_ps, top_p = _sampling_parameter(top_p, "top_p", rows, "float32", lambda x: 0 <= x <= 1)
    min_ps, min_p = _sampling_parameter(min_p, "min_p", rows, "float32", lambda x: 0 <= x <= 1)
    tokens, probabilities = AMDStorage(rows, "int64"), AMDStorage(rows, "float32")
    if rows:
        tokens.runtime.call("qutai_amd_sample", logits.ptr, uniforms.ptr, tokens.ptr, probabilities.ptr, rows, vocab,
                            temperatures, float(temperature), top_ks, top_k, top_ps, float(top_p), min_ps, float(min_p),
                            code(logits.dtype), code(uniforms.dtype))
    return tokens, probabilities


def head_gradient(logits, labels, rows, vocab, gradient, count, *, start=0):
    """In place: logits = g / count * (softmax - onehot) (cuda_lm.py:646-660)."""
    _, pointer = _head_labels(labels, start, rows)
    g = gradient if gradient.dtype == "float32" else amd.from_storage(gradient, dtype="float32")
    if rows:
        logits.runtime.call("qutai_amd_head_gradient", logits.ptr, pointer, g.ptr, rows, vocab, 1.0 / count,
                            code(logits.dtype))
    return logits
