"""Launch wrappers with the names, argument meaning and error behaviour of the reference's Rust
launchers (src/compute/kernels.rs), over the C ABI of libvib3_cuda.so.

Pointers are raw device addresses (ints) or CUDA tensors; ``stream`` is a raw cudaStream_t (int)
and defaults to torch's current stream.  A non-zero launcher return raises Vib3Error, as the
reference maps it to Error::Cuda (kernels.rs:145-150).  There is no CPU path here: the
reference's ``CudaStream::cpu_only()`` fallbacks are restated only in the test oracle."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .core_types import INT4_GROUP_SIZE, SCORING_SIGMOID, SCORING_SOFTMAX, W_F16, W_F32, X_BF16, X_F16, X_F32
from .lib import check, lib


def _ptr(t) -> int:
    if t is None:
        return 0
    if isinstance(t, int):
        return t
    if not t.is_cuda and not t.is_pinned():
        raise ValueError("device tensor (or pinned, device-addressable host tensor) expected")
    return t.data_ptr()


def _stream(stream: Optional[int] = None) -> int:
    """The raw stream given, or torch's current one.  (torch.cuda.current_stream() builds a Stream object through six
    layers of device look-ups: half of the host time of a per-page call.)"""
    if stream is not None:
        return stream
    if not torch.cuda.is_initialized():
        torch.cuda.init()
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def x_dtype_code(t: torch.Tensor) -> int:
    return {torch.float32: X_F32, torch.float16: X_F16, torch.bfloat16: X_BF16}[t.dtype]


def partial_matmul(input, weight_page, output, k: int, m_slice: int, stream: Optional[int] = None) -> None:
    """kernels.rs:25-152, INT4 arm: y_f16[m_slice] = W_page . x_f16; the scales pointer is derived
    from the page pointer exactly as kernels.rs:94-98 does."""
    page = _ptr(weight_page)
    scales = page + ((k + 1) // 2) * m_slice
    check("partial_matmul_int4", lib().vib3_launch_partial_matmul_int4(
        _ptr(input), page, scales, _ptr(output), k, m_slice, INT4_GROUP_SIZE, _stream(stream)))


def partial_matmul_f32(input, weight_page, output, k: int, m_slice: int, stream: Optional[int] = None) -> None:
    """kernels.rs:375-455, INT4 arm: fp32 input, fp16 output."""
    page = _ptr(weight_page)
    scales = page + ((k + 1) // 2) * m_slice
    check("partial_matmul_int4_f32", lib().vib3_launch_partial_matmul_int4_f32(
        _ptr(input), page, scales, _ptr(output), k, m_slice, INT4_GROUP_SIZE, _stream(stream)))


def silu_mul(silu_operand, mul_operand, output, dim: int, stream: Optional[int] = None) -> None:
    check("silu_mul", lib().vib3_launch_silu_mul(_ptr(silu_operand), _ptr(mul_operand), _ptr(output), dim, _stream(stream)))


def partial_swiglu_f32(input, up_page, gate_page, output, hidden_dim: int, m_slice: int,
                       swiglu_temps: Optional[Tuple] = None, stream: Optional[int] = None) -> None:
    """kernels.rs:459-600, INT4 arm.  With temps: the reference's decomposition (two fp32-input
    matmuls rounded to fp16, then silu_mul, kernels.rs:493-541).  Without: the fused kernel
    (cuda_ffi.rs:344-355), one rounding."""
    if swiglu_temps is not None:
        up_tmp, gate_tmp = swiglu_temps
        partial_matmul_f32(input, up_page, up_tmp, hidden_dim, m_slice, stream)
        partial_matmul_f32(input, gate_page, gate_tmp, hidden_dim, m_slice, stream)
        silu_mul(gate_tmp, up_tmp, output, m_slice, stream)
        return
    up, gate = _ptr(up_page), _ptr(gate_page)
    off = ((hidden_dim + 1) // 2) * m_slice
    check("fused_swiglu_int4_f32", lib().vib3_launch_fused_swiglu_int4_f32(
        _ptr(input), up, up + off, gate, gate + off, _ptr(output), hidden_dim, m_slice, INT4_GROUP_SIZE, _stream(stream)))


def weighted_accumulate(output, expert_output, weight: float, dim: int, stream: Optional[int] = None) -> None:
    check("weighted_accumulate", lib().vib3_launch_weighted_accumulate(_ptr(output), _ptr(expert_output), weight, dim, _stream(stream)))


def weighted_accumulate_f32(output, expert_output, weight: float, dim: int, stream: Optional[int] = None) -> None:
    check("weighted_accumulate_f32", lib().vib3_launch_weighted_accumulate_f32(_ptr(output), _ptr(expert_output), weight, dim, _stream(stream)))


def weighted_accumulate_f32_f32(output, expert_output, weight: float, dim: int, stream: Optional[int] = None) -> None:
    check("weighted_accumulate_f32_f32", lib().vib3_launch_weighted_accumulate_f32_f32(_ptr(output), _ptr(expert_output), weight, dim, _stream(stream)))


def residual_add_f32_f32(accumulator, layer_output, dim: int, stream: Optional[int] = None) -> None:
    check("residual_add_f32_f32", lib().vib3_launch_residual_add_f32_f32(_ptr(accumulator), _ptr(layer_output), dim, _stream(stream)))


def rms_norm_f32(input_f32, output_f32, weight_f16, hidden_dim: int, eps: float, stream: Optional[int] = None) -> None:
    """kernels.rs:2560-2603 (GPU arm): fp32 in, fp32 out, fp16 weight."""
    check("rms_norm_f32", lib().vib3_launch_rms_norm_f32(_ptr(input_f32), _ptr(output_f32), _ptr(weight_f16), hidden_dim, eps,
                                                        _stream(stream)))


EXACT_HOLD = 2   # added to a router launch's exact_order: the producer of x lets its dependents start early


_X_TYPES = {torch.float32: (X_F32, 4), torch.float16: (X_F16, 2), torch.bfloat16: (X_BF16, 2)}     # code, bytes


def _row_stride(t: torch.Tensor, shape) -> Optional[int]:
    """From row to row of t, if it has a contiguous row for each of [T, H] (a single one may be a vector); None otherwise."""
    if t.shape == shape or (t.dim() == 2 and t.shape[0] >= shape[0] and t.shape[1] >= shape[1]):
        stride, last = t.stride()
        return stride if last == 1 else None
    return 1 if t.dim() == 1 and shape[0] <= 1 and t.shape[0] >= shape[1] and t.stride(0) == 1 else None


def residual_rms_norm(hidden: torch.Tensor, delta, weight_f16, eps: float, x_out: torch.Tensor, stream: Optional[int] = None,
                      delta2=None, center: bool = False, early_dependents: bool = False) -> None:
    """hidden [T, H] fp32 += delta [T, H] + delta2 [T, H] fp32 (either may be None); x_out [T, H] = cast(rms_norm(hidden) *
    weight) with ``weight_f16`` [H] fp16 or, as a tensor of that type, bf16 (None: no weight): one launch.
    ``early_dependents``: the next launch of the stream may start while this one runs; it must be a router launch with ``EXACT_HOLD`` added to its exact_order argument (see include/vib3_b200.h)."""
    shape = hidden.shape
    if len(shape) != 2 or hidden.dtype != torch.float32 or hidden.stride(1) != 1:
        raise ValueError("hidden: fp32 [T, H] with contiguous rows expected")
    if hidden.is_cuda and hidden.get_device() != _current_device():     # (a launch on another one would read through a foreign context)
        raise ValueError(f"hidden: on the current device (cuda:{_current_device()}) expected, got {hidden.device}")
    # (the launcher knows addresses and strides only: what is smaller than hidden would be written or read behind its end)
    T, H = shape
    x_type, x_stride = _X_TYPES.get(x_out.dtype), _row_stride(x_out, shape)
    if x_type is None or x_stride is None or (T > 1 and x_stride < H):
        raise ValueError("x_out: fp32, fp16 or bf16 with room for hidden's rows, each contiguous, expected")
    d_type, d_stride = (0, 0), 0
    if delta is not None:
        d_type, d_stride = _X_TYPES.get(delta.dtype), _row_stride(delta, shape)
        if d_type is None or d_stride is None:
            raise ValueError("delta: fp32, fp16 or bf16 with a contiguous row for each of hidden's expected")
    d2_stride = 0
    if delta2 is not None:
        d2_stride = _row_stride(delta2, shape)
        if delta2.dtype != torch.float32 or d2_stride is None:
            raise ValueError("delta2: fp32 with a contiguous row for each of hidden's expected")
    flags = int(center) | (2 if early_dependents else 0)
    if isinstance(weight_f16, torch.Tensor):
        w_type = weight_f16.dtype
        if w_type == torch.bfloat16:
            flags |= 4
        elif w_type != torch.float16:
            raise ValueError(f"norm weights: fp16 or bf16 expected, got {w_type}")
        if weight_f16.numel() < H or not weight_f16.is_contiguous():
            raise ValueError("norm weights: contiguous [H] expected")
    err = lib().vib3_launch_residual_rms_norm(
        _ptr(hidden), hidden.stride(0), _ptr(delta), d_type[0], d_stride * d_type[1], _ptr(delta2), d2_stride, _ptr(weight_f16), eps, flags,
        _ptr(x_out), x_type[0], x_stride * x_type[1], H, T, _stream(stream))
    if err:
        check("residual_rms_norm", err)


def router_gemv_f32(hidden_state, router_weights_f16, scores, hidden_dim: int, num_experts: int,
                    stream: Optional[int] = None) -> None:
    check("router_gemv_f32", lib().vib3_launch_router_gemv_f32(_ptr(hidden_state), _ptr(router_weights_f16), _ptr(scores),
                                                              hidden_dim, num_experts, _stream(stream)))


def router_gemv(hidden_state_f16, router_weights_f16, scores, hidden_dim: int, num_experts: int,
                stream: Optional[int] = None) -> None:
    check("router_gemv", lib().vib3_launch_router_gemv(_ptr(hidden_state_f16), _ptr(router_weights_f16), _ptr(scores),
                                                      hidden_dim, num_experts, _stream(stream)))


def run_router_gpu_topk_nosync(hidden_state_f32, router_weights_f16, scores_buf, bias, out_ids, out_weights,
                               hidden_dim: int, num_experts: int, top_k: int, scoring_mode: int,
                               scaling_factor: float, stream: Optional[int] = None) -> None:
    """kernels.rs:1890-1953: results stay on the device."""
    check("router_topk", lib().vib3_launch_router_topk(
        _ptr(hidden_state_f32), _ptr(router_weights_f16), _ptr(scores_buf), _ptr(bias), _ptr(out_ids), _ptr(out_weights),
        hidden_dim, num_experts, top_k, scoring_mode, scaling_factor, _stream(stream)))


def run_router_gpu_topk(hidden_state_f32, router_weights_f16, scores_buf, bias, out_ids, out_weights, hidden_dim: int,
                        num_experts: int, top_k: int, scoring_mode: int, scaling_factor: float,
                        stream: Optional[int] = None):
    """kernels.rs:1811-1873: launch, synchronise, two small D2H copies -> [(expert, weight)]."""
    run_router_gpu_topk_nosync(hidden_state_f32, router_weights_f16, scores_buf, bias, out_ids, out_weights, hidden_dim,
                               num_experts, top_k, scoring_mode, scaling_factor, stream)
    torch.cuda.current_stream().synchronize()
    ids = out_ids[:top_k].cpu().view(torch.int16).numpy().view("uint16")
    ws = out_weights[:top_k].cpu().numpy()
    return [(int(i), float(w)) for i, w in zip(ids, ws)]


def router_topk_ex(x: torch.Tensor, W: torch.Tensor, scores_buf, bias, out_ids, out_weights, top_k: int,
                   scoring_mode: int, scaling_factor: float, normalize: bool, exact_order: bool, workspace,
                   stream: Optional[int] = None, logit_offset=None) -> None:
    """Single-launch router for fp16/bf16/fp32 activations and fp16/fp32 weights."""
    E, H = W.shape
    w_dtype = {torch.float16: W_F16, torch.float32: W_F32}[W.dtype]
    check("router_topk_ex", lib().vib3_launch_router_topk_ex(
        _ptr(x), x_dtype_code(x), _ptr(W), w_dtype, _ptr(scores_buf), _ptr(bias), _ptr(logit_offset), _ptr(out_ids),
        _ptr(out_weights), H, E,
        top_k, scoring_mode, scaling_factor, int(normalize), int(exact_order), _ptr(workspace), _stream(stream)))


def router_topk_batch(xs: torch.Tensor, W: torch.Tensor, scores_buf: torch.Tensor, bias, logit_offset, out_ids: torch.Tensor,
                      out_weights: torch.Tensor, top_k: int, scoring_mode: int, scaling_factor: float, normalize: bool,
                      exact_order: bool, workspace: torch.Tensor, stream: Optional[int] = None) -> None:
    """The router for T tokens in ONE call (the weights are read once): xs [T, H]; scores_buf [T, 3E] fp32,
    out_ids [T, >= top_k] int16, out_weights [T, >= top_k] fp32, workspace [T, 4] int32 (zero before the first call)."""
    E, H = W.shape
    T = xs.shape[0]
    w_dtype = {torch.float16: W_F16, torch.float32: W_F32}[W.dtype]
    check("router_topk_batch", lib().vib3_launch_router_topk_batch(
        _ptr(xs), x_dtype_code(xs), xs.stride(0) * xs.element_size(), T, _ptr(W), w_dtype, _ptr(scores_buf),
        scores_buf.stride(0), _ptr(bias), _ptr(logit_offset), _ptr(out_ids), out_ids.stride(0), _ptr(out_weights),
        out_weights.stride(0), H, E, top_k, scoring_mode, scaling_factor, int(normalize), int(exact_order), _ptr(workspace),
        _stream(stream)))


def moe_layer_int4_paged(x: torch.Tensor, page_table: int, num_experts: int, shared_pages: int, expert_ids,
                         expert_weights, top_k: int, shared_weight: float, act_scratch, out, out_accumulate: bool,
                         hidden_dim: int, expert_hidden_dim: int, pages_per_segment: int, rows_per_page_gate_up: int,
                         rows_per_page_down: int, status=None, stream: Optional[int] = None, phase: int = 3) -> None:
    """phase 3: both launches; 1: gate/up + SiLU only; 2: down + accumulate only."""
    fn = {3: lib().vib3_launch_moe_layer_int4_paged, 1: lib().vib3_launch_moe_gate_up_int4_paged,
          2: lib().vib3_launch_moe_down_int4_paged}[phase]
    check("moe_layer_int4_paged", fn(
        _ptr(x), x_dtype_code(x), page_table, num_experts, shared_pages or 0, _ptr(expert_ids), _ptr(expert_weights), top_k,
        shared_weight, _ptr(act_scratch), _ptr(out), int(out_accumulate), hidden_dim, expert_hidden_dim,
        pages_per_segment, rows_per_page_gate_up, rows_per_page_down, INT4_GROUP_SIZE, _ptr(status), _stream(stream)))


def moe_layer_routed_int4_paged(x: torch.Tensor, router_w: torch.Tensor, scores_buf, bias, logit_offset, ids_out, weights_out,
                                top_k: int, scoring_mode: int, scaling_factor: float, normalize: bool, exact_order: bool,
                                workspace, page_table: int, num_experts: int, shared_pages: int, shared_weight: float,
                                act_scratch, out, out_accumulate: bool, hidden_dim: int, expert_hidden_dim: int,
                                pages_per_segment: int, rows_per_page_gate_up: int, rows_per_page_down: int, status=None,
                                stream: Optional[int] = None) -> None:
    """Router and experts of one token; the routing (ids_out, weights_out) is an output.  Two launches where
    the gate/up kernel can route the token in its own prologue, three otherwise."""
    w_dtype = {torch.float16: W_F16, torch.float32: W_F32}[router_w.dtype]
    check("moe_layer_routed_int4_paged", lib().vib3_launch_moe_layer_routed_int4_paged(
        _ptr(x), x_dtype_code(x), _ptr(router_w), w_dtype, _ptr(scores_buf), _ptr(bias), _ptr(logit_offset), _ptr(ids_out),
        _ptr(weights_out), num_experts, top_k, scoring_mode, scaling_factor, int(normalize), int(exact_order), _ptr(workspace),
        page_table, shared_pages or 0, shared_weight, _ptr(act_scratch), _ptr(out), int(out_accumulate), hidden_dim,
        expert_hidden_dim, pages_per_segment, rows_per_page_gate_up, rows_per_page_down, INT4_GROUP_SIZE, _ptr(status),
        _stream(stream)))


def moe_layer_int4_paged_var(x: torch.Tensor, page_table: int, num_experts: int, shared_pages: int, expert_ids,
                             expert_weights, top_k: int, shared_weight: float, act_scratch, out, out_accumulate: bool,
                             hidden_dim: int, expert_hidden_dim: int, pages_per_segment: int,
                             rows_per_page_gate_up: int, rows_per_page_down: int, num_active_dev, status=None,
                             stream: Optional[int] = None) -> None:
    """The fused sublayer over the first min(top_k, *num_active_dev) routed slots (device-side count)."""
    check("moe_layer_int4_paged_var", lib().vib3_launch_moe_layer_int4_paged_var(
        _ptr(x), x_dtype_code(x), page_table, num_experts, shared_pages or 0, _ptr(expert_ids), _ptr(expert_weights), top_k,
        shared_weight, _ptr(act_scratch), _ptr(out), int(out_accumulate), hidden_dim, expert_hidden_dim,
        pages_per_segment, rows_per_page_gate_up, rows_per_page_down, INT4_GROUP_SIZE, _ptr(status), _stream(stream),
        _ptr(num_active_dev)))


def moe_layer_int4_paged_grouped(x, x_dtype: int, x_stride_bytes: int, n_tokens: int, page_table: int, num_experts: int,
                                 shared_pages: int, shared_token: int, pair_experts, pair_weights, pair_tokens,
                                 pair_capacity: int, pair_begin: int, num_pairs_dev, shared_weight: float, act_scratch, out,
                                 out_stride: int, out_accumulate: bool, hidden_dim: int, expert_hidden_dim: int,
                                 pages_per_segment: int, rows_per_page_gate_up: int, rows_per_page_down: int, status=None,
                                 stream: Optional[int] = None) -> None:
    """One launch pair over the (token, expert) pairs of several tokens (expert parallelism)."""
    check("moe_layer_int4_paged_grouped", lib().vib3_launch_moe_layer_int4_paged_grouped(
        _ptr(x), x_dtype, x_stride_bytes, n_tokens, page_table, num_experts, shared_pages or 0, shared_token,
        _ptr(pair_experts), _ptr(pair_weights), _ptr(pair_tokens), pair_capacity, pair_begin, _ptr(num_pairs_dev),
        shared_weight, _ptr(act_scratch), _ptr(out), out_stride, int(out_accumulate), hidden_dim, expert_hidden_dim,
        pages_per_segment, rows_per_page_gate_up, rows_per_page_down, INT4_GROUP_SIZE, _ptr(status), _stream(stream)))


def select_local_pairs(ids, ids_stride_bytes: int, weights, weights_stride_bytes: int, n_tokens: int, top_k: int,
                       expert_lo: int, expert_hi: int, pair_experts, pair_weights, pair_tokens, capacity: int, count_out,
                       stream: Optional[int] = None) -> None:
    check("select_local_pairs", lib().vib3_launch_select_local_pairs(
        _ptr(ids), ids_stride_bytes, _ptr(weights), weights_stride_bytes, n_tokens, top_k, expert_lo, expert_hi,
        _ptr(pair_experts), _ptr(pair_weights), _ptr(pair_tokens), capacity, _ptr(count_out), _stream(stream)))


def moe_layer_step_host(x_host: torch.Tensor, x_dev: torch.Tensor, router_w: torch.Tensor, scores_buf, bias, ids_dev, weights_dev,
                        num_experts: int, top_k: int, scoring_mode: int, scaling_factor: float, normalize: bool,
                        exact_order: bool, workspace, page_table: int, shared_pages: int, shared_weight: float, act_scratch,
                        out_dev, out_host: torch.Tensor, hidden_dim: int, expert_hidden_dim: int, pages_per_segment: int,
                        rows_per_page_gate_up: int, rows_per_page_down: int, status=None, stream: Optional[int] = None) -> None:
    """One token from and to host memory through one C call (copy in, router, experts, synchronise)."""
    w_dtype = {torch.float16: W_F16, torch.float32: W_F32}[router_w.dtype]
    if x_host.is_cuda or out_host.is_cuda:
        raise ValueError("host tensors expected")
    if out_dev is None and not out_host.is_pinned():
        raise ValueError("out_host must be pinned when no device output buffer is given")
    check("moe_layer_step_host", lib().vib3_moe_layer_step_host(
        x_host.data_ptr(), x_dtype_code(x_host), _ptr(x_dev), _ptr(router_w), w_dtype, _ptr(scores_buf), _ptr(bias), _ptr(ids_dev),
        _ptr(weights_dev), num_experts, top_k, scoring_mode, scaling_factor, int(normalize), int(exact_order), _ptr(workspace),
        page_table, shared_pages or 0, shared_weight, _ptr(act_scratch), _ptr(out_dev), out_host.data_ptr(), hidden_dim,
        expert_hidden_dim, pages_per_segment, rows_per_page_gate_up, rows_per_page_down, INT4_GROUP_SIZE, _ptr(status),
        _stream(stream)))


def sum_rows_f32(rows_in: torch.Tensor, out: torch.Tensor, stream: Optional[int] = None) -> None:
    """out[c] = sum_r rows_in[r, c], rows added in order."""
    check("sum_rows_f32", lib().vib3_launch_sum_rows_f32(_ptr(rows_in), rows_in.shape[0], rows_in.shape[1], rows_in.stride(0),
                                                         _ptr(out), _stream(stream)))


def peer_publish(src: torch.Tensor, src_stride_bytes: int, nbytes: int, dst_table: torch.Tensor, dst_stride_bytes: int,
                 flag_table: torch.Tensor, step_counter: torch.Tensor, step_offset: int, rank: int, world: int,
                 stream: Optional[int] = None) -> None:
    """Store nbytes from src (+ d * src_stride_bytes) into every rank d's buffer at slot `rank`, then the flag
    (*step_counter + step_offset)."""
    check("peer_publish", lib().vib3_launch_peer_publish(_ptr(src), src_stride_bytes, nbytes, _ptr(dst_table), dst_stride_bytes,
                                                         _ptr(flag_table), _ptr(step_counter), step_offset, rank, world, _stream(stream)))


def peer_publish_rows(src: torch.Tensor, add_src: torch.Tensor, row_bytes: int, add_count: torch.Tensor, add_threshold: int,
                      dst_table: torch.Tensor, dst_stride_bytes: int, flag_table: torch.Tensor, step_counter: torch.Tensor,
                      step_offset: int, rank: int, world: int, stream: Optional[int] = None) -> None:
    """peer_publish of fp32 rows: rank d receives src[d] + (add_src[d] if *add_count > add_threshold)."""
    check("peer_publish_rows", lib().vib3_launch_peer_publish_rows(
        _ptr(src), _ptr(add_src), src.stride(0) * 4, row_bytes, _ptr(add_count), add_threshold, _ptr(dst_table), dst_stride_bytes,
        _ptr(flag_table), _ptr(step_counter), step_offset, rank, world, _stream(stream)))


def peer_wait(flags: torch.Tensor, step_counter: torch.Tensor, world: int, advance: bool, status, stream: Optional[int] = None) -> None:
    """Wait (bounded) until every peer's flag has reached the next step; advance the step counter."""
    check("peer_wait", lib().vib3_launch_peer_wait(_ptr(flags), _ptr(step_counter), world, int(advance), _ptr(status), _stream(stream)))


def peer_select_pairs(flags, step_counter, world: int, status, ids, ids_stride_bytes: int, weights, weights_stride_bytes: int,
                      top_k: int, expert_lo: int, expert_hi: int, pair_experts, pair_weights, pair_tokens, capacity: int, count_out,
                      stream: Optional[int] = None) -> None:
    """peer_wait for the messages (advancing the step) and select_local_pairs over them in one launch."""
    check("peer_select_pairs", lib().vib3_launch_peer_select_pairs(
        _ptr(flags), _ptr(step_counter), world, _ptr(status), _ptr(ids), ids_stride_bytes, _ptr(weights), weights_stride_bytes, top_k,
        expert_lo, expert_hi, _ptr(pair_experts), _ptr(pair_weights), _ptr(pair_tokens), capacity, _ptr(count_out), _stream(stream)))


def peer_sum_rows(flags, step_counter, world: int, status, rows_in: torch.Tensor, out: torch.Tensor, stream: Optional[int] = None) -> None:
    """Wait for the partial rows of the current step, then out[c] = sum_r rows_in[r, c] in row order: one launch."""
    check("peer_sum_rows", lib().vib3_launch_peer_sum_rows(_ptr(flags), _ptr(step_counter), world, _ptr(status), _ptr(rows_in),
                                                           rows_in.shape[0], rows_in.shape[1], rows_in.stride(0), _ptr(out), _stream(stream)))


def select_local_experts(ids, weights, top_k: int, expert_lo: int, expert_hi: int, ids_out, weights_out, count_out,
                         stream: Optional[int] = None) -> None:
    check("select_local_experts", lib().vib3_launch_select_local_experts(
        _ptr(ids), _ptr(weights), top_k, expert_lo, expert_hi, _ptr(ids_out), _ptr(weights_out), _ptr(count_out),
        _stream(stream)))


# ── latent attention ─────────────────────────────────────────────────────────────────────────
# (One look at a tensor's shape, strides and dtype each: a decode step makes four of these calls per layer, and what a launch takes
# on the device is less than ten such looks.)

LATENT_RANK, LATENT_ROPE = 512, 64
LATENT_ROW = LATENT_RANK + LATENT_ROPE
_X_CODES = {torch.float32: X_F32, torch.float16: X_F16, torch.bfloat16: X_BF16}
_I32, _I64, _F32, _F64 = torch.int32, torch.int64, torch.float32, torch.float64


_current_device, _current_stream = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)
_latent = None       # the library's latent launchers, once the device is there


def _bind_latent():
    """(append, query, value, attention): the launchers, looked up once.  CUDA is initialised here, not by every call."""
    global _latent
    if not torch.cuda.is_initialized():
        torch.cuda.init()
    h = lib()
    _latent = (h.vib3_launch_latent_append_paged, h.vib3_launch_latent_query, h.vib3_launch_latent_value, h.vib3_launch_latent_attention_paged)
    return _latent


def _foreign(*tensors) -> ValueError:
    return ValueError(f"operands have to be on the current device (cuda:{_current_device()}), got {[str(t.device) for t in tensors if t is not None]}")


def latent_append(kv: torch.Tensor, norm_weight: Optional[torch.Tensor], eps: float, positions: torch.Tensor, slots: torch.Tensor,
                  inv_freq: torch.Tensor, cache: torch.Tensor, pairs: bool = True, rope_scale: float = 1.0,
                  status: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> None:
    """Rows of latent attention into the paged cache (the reference's MLA cache append, cuda/src/kernels.cu:1709, for T tokens):
    kv [T, 576] fp32 / fp16 / bf16 -> cache [pages, page_size, 576] fp16 / bf16 at ``slots`` [T] int64 (page * page_size + row;
    negative: skipped), the first 512 values RMS-normalised with ``norm_weight`` [512] (the cache's dtype; None: not
    normalised), the other 64 rotated by ``positions`` [T] int32 * ``inv_freq`` [32] float64.  ``pairs``: neighbouring values
    turn together (else values 32 apart).  ``status`` [1] int32 receives VIB3_STATUS_MISSING_PAGE for a slot beyond the cache."""
    (T, W), (kv_stride, k1) = kv.shape, kv.stride()
    (pages, page, R), (page_stride, row_stride, c1) = cache.shape, cache.stride()
    code, dt = _X_CODES.get(kv.dtype), cache.dtype
    if W != LATENT_ROW or k1 != 1 or code is None:
        raise ValueError("kv: fp32, fp16 or bf16 [T, 576] with contiguous rows expected")
    if R != LATENT_ROW or c1 != 1 or (dt != torch.bfloat16 and dt != torch.float16):
        raise ValueError("cache: fp16 or bf16 [pages, page_size, 576] with contiguous rows expected")
    if slots.shape != (T,) or slots.dtype != _I64 or not slots.is_contiguous():
        raise ValueError("slots: contiguous int64 [T] expected")
    if positions.shape != (T,) or positions.dtype != _I32 or not positions.is_contiguous():
        raise ValueError("positions: contiguous int32 [T] expected")
    if inv_freq.shape != (LATENT_ROPE // 2,) or inv_freq.dtype != _F64 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq: contiguous float64 [32] expected")
    if norm_weight is not None and (norm_weight.shape != (LATENT_RANK,) or norm_weight.dtype != dt or not norm_weight.is_contiguous()):
        raise ValueError("norm_weight: contiguous [512] of the cache's dtype expected")
    if status is not None and (status.dtype != _I32 or status.numel() == 0):
        raise ValueError("status: int32 [1] expected")
    launch = (_latent or _bind_latent())[0]
    dev = _current_device()     # (a launch on another one would read through a foreign context)
    if not (dev == kv.get_device() == cache.get_device() == slots.get_device() == positions.get_device() == inv_freq.get_device()
            == (kv if norm_weight is None else norm_weight).get_device() == (kv if status is None else status).get_device()):
        raise _foreign(kv, cache, slots, positions, inv_freq, norm_weight, status)
    err = launch(
        kv.data_ptr(), code, kv_stride, 0 if norm_weight is None else norm_weight.data_ptr(), eps, positions.data_ptr(), slots.data_ptr(),
        inv_freq.data_ptr(), rope_scale, 1 if pairs else 0, T, cache.data_ptr(), _X_CODES[dt], pages, page, page_stride, row_stride,
        0 if status is None else status.data_ptr(), _current_stream(dev) if stream is None else stream)
    if err:
        check("latent_append", err)


def latent_query(q: torch.Tensor, w_uk: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, out: torch.Tensor,
                 pairs: bool = True, rope_scale: float = 1.0, status: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> None:
    """The heads' queries in the latent space (cuda/src/kernels.cu:1679 for T tokens): q [T, H, nope + 64], w_uk [H, nope, 512] ->
    out [T, H, 576] = (q[..., :nope] . w_uk, q[..., nope:] rotated).  One 16-bit dtype; w_uk may be a view of [H, nope + value, 512].
    ``status`` [1] int32 receives VIB3_STATUS_TIMEOUT."""
    (T, H, width), (q0, q1, q2) = q.shape, q.stride()
    (heads, nope, R), (w0, w1, w2) = w_uk.shape, w_uk.stride()
    o0, o1, o2 = out.stride()
    dt = q.dtype
    if width != nope + LATENT_ROPE or heads != H or q2 != 1:
        raise ValueError("q: [T, H, nope + 64] with contiguous rows expected")
    if R != LATENT_RANK or w2 != 1 or w1 != LATENT_RANK:
        raise ValueError("w_uk: [H, nope, 512] with contiguous heads expected")
    if out.shape != (T, H, LATENT_ROW) or o2 != 1:
        raise ValueError("out: [T, H, 576] with contiguous rows expected")
    if positions.shape != (T,) or positions.dtype != _I32 or not positions.is_contiguous():
        raise ValueError("positions: contiguous int32 [T] expected")
    if inv_freq.shape != (LATENT_ROPE // 2,) or inv_freq.dtype != _F64 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq: contiguous float64 [32] expected")
    if (dt != torch.bfloat16 and dt != torch.float16) or w_uk.dtype != dt or out.dtype != dt:
        raise ValueError("one dtype, fp16 or bf16, expected")
    if status is not None and (status.dtype != _I32 or status.numel() == 0):
        raise ValueError("status: int32 [1] expected")
    launch = (_latent or _bind_latent())[1]
    dev = _current_device()     # (a launch on another one would read through a foreign context)
    if not (dev == q.get_device() == w_uk.get_device() == positions.get_device() == inv_freq.get_device() == out.get_device()
            == (q if status is None else status).get_device()):
        raise _foreign(q, w_uk, positions, inv_freq, out, status)
    err = launch(
        q.data_ptr(), q0, q1, w_uk.data_ptr(), w0, positions.data_ptr(), inv_freq.data_ptr(), rope_scale, 1 if pairs else 0, out.data_ptr(),
        o0, o1, T, H, nope, _X_CODES[dt], 0 if status is None else status.data_ptr(), _current_stream(dev) if stream is None else stream)
    if err:
        check("latent_query", err)


def latent_value(o: torch.Tensor, w_uv: torch.Tensor, out: torch.Tensor, status: Optional[torch.Tensor] = None,
                 stream: Optional[int] = None) -> None:
    """The heads' outputs from their weighted latents (cuda/src/kernels.cu:1624 for T tokens): o [T, H, 512], w_uv [H, value, 512] ->
    out [T, H, value].  One 16-bit dtype.  ``status`` [1] int32 receives VIB3_STATUS_TIMEOUT."""
    (T, H, width), (i0, i1, i2) = o.shape, o.stride()
    (heads, value, R), (w0, w1, w2) = w_uv.shape, w_uv.stride()
    o0, o1, o2 = out.stride()
    dt = o.dtype
    if width != LATENT_RANK or i2 != 1 or heads != H:
        raise ValueError("o: [T, H, 512] with contiguous rows expected")
    if R != LATENT_RANK or w2 != 1 or w1 != LATENT_RANK:
        raise ValueError("w_uv: [H, value, 512] with contiguous heads expected")
    if out.shape != (T, H, value) or o2 != 1:
        raise ValueError("out: [T, H, value] with contiguous rows expected")
    if (dt != torch.bfloat16 and dt != torch.float16) or w_uv.dtype != dt or out.dtype != dt:
        raise ValueError("one dtype, fp16 or bf16, expected")
    if status is not None and (status.dtype != _I32 or status.numel() == 0):
        raise ValueError("status: int32 [1] expected")
    launch = (_latent or _bind_latent())[2]
    dev = _current_device()     # (a launch on another one would read through a foreign context)
    if not (dev == o.get_device() == w_uv.get_device() == out.get_device() == (o if status is None else status).get_device()):
        raise _foreign(o, w_uv, out, status)
    err = launch(o.data_ptr(), i0, i1, w_uv.data_ptr(), w0, out.data_ptr(), o0, o1, T, H, value, _X_CODES[dt],
                 0 if status is None else status.data_ptr(), _current_stream(dev) if stream is None else stream)
    if err:
        check("latent_value", err)


def latent_attention_workspace_bytes() -> int:
    return lib().vib3_latent_attention_workspace_bytes()


def latent_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                     out: torch.Tensor, lse: Optional[torch.Tensor] = None, *, workspace: torch.Tensor,
                     status: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> None:
    """Attention in the latent space over the paged cache (cuda/src/kernels.cu:1570 for the newest tokens of a batch): q [B * q_len,
    H, 576] (sequence b's q_len tokens together), cache [pages, page_size, 576], page_table [B, max_pages] int32, seq_lens [B] int32
    (keys of each sequence, its new tokens included) -> out [B * q_len, H, 512] and, if given, lse [B * q_len, H] fp32.  Token j of
    a sequence sees the keys up to position seq_lens - q_len + j; a row that sees none is 0 and -inf.  Rows of the cache behind a length
    may hold anything, those within it have to be finite.  ``workspace``: a uint8
    tensor of latent_attention_workspace_bytes(), not shared by calls that may overlap."""
    (T, H, width), (q0, q1, q2) = q.shape, q.stride()
    (pages, page, R), (c0, c1, c2) = cache.shape, cache.stride()
    (B, max_pages), (t0, t1) = page_table.shape, page_table.stride()
    o0, o1, o2 = out.stride()
    dt = q.dtype
    q_len = T // B if B else 0
    if width != LATENT_ROW or q2 != 1 or q_len * B != T:
        raise ValueError("q: [B * q_len, H, 576] with contiguous rows expected")
    if R != LATENT_ROW or c2 != 1:
        raise ValueError("cache: [pages, page_size, 576] with contiguous rows expected")
    if page_table.dtype != _I32 or (t1 != 1 and max_pages > 1):
        raise ValueError("page_table: int32 [B, max_pages] with contiguous rows expected")
    if seq_lens.shape != (B,) or seq_lens.dtype != _I32 or not seq_lens.is_contiguous():
        raise ValueError("seq_lens: contiguous int32 [B] expected")
    if out.shape != (T, H, LATENT_RANK) or o2 != 1:
        raise ValueError("out: [B * q_len, H, 512] with contiguous rows expected")
    if lse is not None and (lse.shape != (T, H) or lse.dtype != _F32 or not lse.is_contiguous()):
        raise ValueError("lse: contiguous fp32 [B * q_len, H] expected")
    if (dt != torch.bfloat16 and dt != torch.float16) or cache.dtype != dt or out.dtype != dt:
        raise ValueError("one dtype, fp16 or bf16, expected")
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace: contiguous uint8 expected")
    if status is not None and (status.dtype != _I32 or status.numel() == 0):
        raise ValueError("status: int32 [1] expected")
    launch = (_latent or _bind_latent())[3]
    dev = _current_device()     # (a launch on another one would read through a foreign context)
    if not (dev == q.get_device() == cache.get_device() == page_table.get_device() == seq_lens.get_device() == out.get_device()
            == workspace.get_device() == (q if lse is None else lse).get_device() == (q if status is None else status).get_device()):
        raise _foreign(q, cache, page_table, seq_lens, out, workspace, lse, status)
    err = launch(
        q.data_ptr(), q0, q1, cache.data_ptr(), pages, page, c0, c1, page_table.data_ptr(), t0, max_pages, seq_lens.data_ptr(), B, q_len, H,
        scale, _X_CODES[dt], out.data_ptr(), o0, o1, 0 if lse is None else lse.data_ptr(), workspace.data_ptr(), workspace.numel(),
        0 if status is None else status.data_ptr(), _current_stream(dev) if stream is None else stream)
    if err:
        check("latent_attention", err)


__all__ = [n for n in dir() if not n.startswith("_")] + ["SCORING_SOFTMAX", "SCORING_SIGMOID"]
