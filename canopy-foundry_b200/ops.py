"""Operator mirror of the reference's FP8 / MoE interface on torch CUDA tensors.

Function names, argument order and meaning follow include/ida_native/kernels.hpp:983-1052 (FP8),
:313-423 (MoE) and the file-static helpers of src/trainer.cu (lt_gemm_fp8_nt :4498, fp8_quant_act
:4732, refresh_fp8_weights :4694). torch supplies device memory and streams only; every operator
runs in libcanopy_fp8.so on the current torch stream. A failing call raises CanopyError, where the
reference throws std::runtime_error.
"""
import ctypes as C

import torch

from . import _capi
from ._capi import E4M3_MAX, E5M2_MAX, CanopyError, check

__all__ = [
    "E4M3_MAX", "E5M2_MAX", "CanopyError", "Fp8Ctx", "ActSlot", "Fp8Weight",
    "fp8_amax_bf16", "fp8_scale_from_amax", "fp8_quantize_e4m3", "fp8_quantize_e5m2",
    "fp8_quantize_e4m3_record", "fp8_quantize_e5m2_record", "fp8_update_delayed_scale",
    "fp8_quantize_transpose_e4m3", "fp8_quant_and_transpose_e4m3", "transpose_u8", "fp8_clip_probe",
    "fp8_elem_clip_count", "fp8_pack_bf16_e4m3_raw", "fp8_pack_bf16_e4m3_raw_and_dequant",
    "fp8_unpack_e4m3_raw_bf16", "lt_gemm_fp8_nt", "gemm_fp8_nn", "gemm_fp8_nn_grouped", "lt_gemm_fp8_tn_accum_f32", "gemm_fp8_dw_accum", "gemm_fp8_nt_reduce_scatter", "f32_to_bf16_and_zero", "gemm_fp8_nt_grouped", "gemm_fp8_nt_segments", "gemm_fp8_nt_segments_scatter",
    "fp8_quant_act", "fp8_swiglu_quant_act", "gemm_fp8_swiglu_quant_act", "fp8_interleave_gate_up", "refresh_fp8_weight", "fp8_linear_forward", "bias_add_strided_bf16", "swiglu_forward",
    "gelu_forward", "lion_step", "lion_step_quantize", "fp8_quantize_rowwise_e4m3", "fp8_quantize_rowwise_given_amax_e4m3", "gemm_fp8_swiglu_bf16_rowamax", "interleave_gate_up_vector", "swiglu_mlp_fp8_rowwise_fused", "swiglu_quantize_rowwise_e4m3", "swiglu_quantize_e4m3_record",
    "rmsnorm_forward", "rmsnorm_quantize_e4m3_record", "rmsnorm_quantize_rowwise_e4m3", "fp8_rmsnorm_quant_act", "rmsnorm_clip_forward", "rmsnorm_clip_quantize_e4m3_record", "fp8_rmsnorm_clip_quant_act",
    "moe_topk_route_f32", "moe_build_expert_row_lists", "moe_expert_offsets_from_counts",
    "moe_gather_rows_u8", "moe_gather_rows_bf16", "moe_scatter_accumulate_rows_bf16",
    "moe_scale_accumulate_bf16", "moe_gather_all_u8", "moe_combine_all_bf16", "moe_combine_sorted_bf16", "moe_expand_route_replicas", "moe_route_dispatch_lists", "moe_route_dispatch_scratch_ints", "moe_ep_plan", "gemm_fp8_nt_grouped_return", "moe_send_row_runs", "peer_barrier", "peer_share_i32", "ROW_RUN_BYTES",
    "block128_row_descale", "fp8_quantize_block128", "swiglu_quantize_block128", "swiglu_backward_quantize_block128", "fp8_quantize_block128x128",
    "add_rmsnorm_quantize_block128", "add_rmsnorm_backward", "add_rmsnorm_backward_scratch_floats",
    "gemm_fp8_block128_nt", "gemm_fp8_block128_nt_grouped", "gemm_fp8_block128_nn", "gemm_fp8_block128_dw",
    "moe_grouped_expert_forward_fp8", "launch_count", "swiglu_mlp_fp8_rowwise", "MoeSwigluFp8", "FfnSwigluFp8", "Fp8Block128Weight", "FfnSwigluFp8Block128",
]


def _s():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t):
    if t is None:
        return None
    assert t.is_cuda, "device tensor expected"
    return C.c_void_p(t.data_ptr())


def _L():
    return _capi.lib()


_rt = None


def _cudart():
    """The CUDA runtime torch already loaded (used only for debug read-backs of slot scalars)."""
    global _rt
    if _rt is None:
        for name in ("libcudart.so.12", "libcudart.so.13", "libcudart.so"):
            try:
                _rt = C.CDLL(name)
                break
            except OSError:
                continue
        if _rt is None:
            raise ImportError("libcudart not found")
        _rt.cudaMemcpy.restype = C.c_int
    return _rt


def launch_count():
    return int(_L().cf_launch_count())


# ---------------------------------------------------------------- quantize / cast
def fp8_amax_bf16(x, amax):
    check(_L().cf_fp8_amax_bf16(_p(x), x.numel(), _p(amax), _s()))


def fp8_scale_from_amax(amax, fp8_max, scale, descale):
    check(_L().cf_fp8_scale_from_amax(_p(amax), fp8_max, _p(scale), _p(descale), _s()))


def fp8_quantize_e4m3(x, out, scale, n=None):
    check(_L().cf_fp8_quantize_e4m3(_p(x), _p(out), _p(scale), x.numel() if n is None else n, _s()))


def fp8_quantize_e5m2(x, out, scale, n=None):
    check(_L().cf_fp8_quantize_e5m2(_p(x), _p(out), _p(scale), x.numel() if n is None else n, _s()))


def fp8_quantize_e4m3_record(x, out, scale, amax, n=None):
    check(_L().cf_fp8_quantize_e4m3_record(_p(x), _p(out), _p(scale), _p(amax), x.numel() if n is None else n, _s()))


def fp8_quantize_e5m2_record(x, out, scale, amax, n=None):
    check(_L().cf_fp8_quantize_e5m2_record(_p(x), _p(out), _p(scale), _p(amax), x.numel() if n is None else n, _s()))


def fp8_update_delayed_scale(amax, fp8_max, scale, descale, history, history_len, cursor, count):
    check(_L().cf_fp8_update_delayed_scale(_p(amax), fp8_max, _p(scale), _p(descale), _p(history), history_len,
                                           _p(cursor), _p(count), _s()))


def fp8_quantize_transpose_e4m3(w, out, scale, K, N):
    check(_L().cf_fp8_quantize_transpose_e4m3(_p(w), _p(out), _p(scale), K, N, _s()))


def fp8_quant_and_transpose_e4m3(x, act8, snap, scale, K, N):
    check(_L().cf_fp8_quant_and_transpose_e4m3(_p(x), _p(act8), _p(snap), _p(scale), K, N, _s()))


def transpose_u8(src, dst, rows, cols):
    check(_L().cf_transpose_u8(_p(src), _p(dst), rows, cols, _s()))


def fp8_clip_probe(amax, scale, fp8_max, stats):
    check(_L().cf_fp8_clip_probe(_p(amax), _p(scale), fp8_max, _p(stats), _s()))


def fp8_elem_clip_count(x, scale, fp8_max, out):
    check(_L().cf_fp8_elem_clip_count(_p(x), _p(scale), fp8_max, x.numel(), _p(out), _s()))


def fp8_pack_bf16_e4m3_raw(x, out, amax, scale, descale, bad_count):
    check(_L().cf_fp8_pack_bf16_e4m3_raw(_p(x), _p(out), _p(amax), _p(scale), _p(descale), _p(bad_count), x.numel(), _s()))


def fp8_pack_bf16_e4m3_raw_and_dequant(x, out, dequant, amax, scale, descale, bad_count):
    check(_L().cf_fp8_pack_bf16_e4m3_raw_and_dequant(_p(x), _p(out), _p(dequant), _p(amax), _p(scale), _p(descale),
                                                     _p(bad_count), x.numel(), _s()))


def fp8_unpack_e4m3_raw_bf16(codes, descale, out):
    check(_L().cf_fp8_unpack_e4m3_raw_bf16(_p(codes), _p(descale), _p(out), codes.numel(), _s()))


# ---------------------------------------------------------------- context, slots
class Fp8Ctx:
    """Counterpart of the reference's Fp8Ctx (src/trainer.cu:3296-3345): owns the shared act8 scratch,
    the scalar pool ActSlots live in and the status word of the tensor-core kernels."""

    def __init__(self, act8_bytes=0):
        h = C.c_void_p()
        check(_L().cf_ctx_create(C.byref(h), act8_bytes))
        self.handle = h
        self.act8_bytes = act8_bytes

    def act8_ptr(self):
        return _L().cf_ctx_act8(self.handle)

    def reserve_workspace(self, nbytes):
        check(_L().cf_ctx_reserve_workspace(self.handle, nbytes))

    def poll_status(self):
        """Synchronises the current stream; raises CanopyError(CF_ERR_DEVICE_WAIT) if a kernel gave up a wait."""
        check(_L().cf_ctx_poll_status(self.handle, _s()))

    def selftest_bounded_wait(self, limit_ms=5):
        """Launches the wait that is designed to run out; the following poll_status() raises CF_ERR_DEVICE_WAIT."""
        check(_L().cf_ctx_selftest_bounded_wait(self.handle, limit_ms, _s()))

    def close(self):
        if self.handle:
            _L().cf_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class ActSlot:
    """Delayed-scaling state of one activation/gradient call site (ActSlot, src/trainer.cu:3248-3279)."""

    def __init__(self, ctx, fp8_max=E4M3_MAX, calib_calls=0):
        self.ctx = ctx
        self.c = _capi.ActSlotStruct()
        check(_L().cf_act_slot_init(ctx.handle, C.byref(self.c), fp8_max, calib_calls, _s()))

    def _read(self, ptr, dtype=torch.float32, n=1):
        """Debug read-back of slot scalars (device pointers owned by the context's pool)."""
        torch.cuda.current_stream().synchronize()
        host = torch.empty(n, dtype=dtype)
        rc = _cudart().cudaMemcpy(C.c_void_p(host.data_ptr()), C.c_void_p(ptr), C.c_size_t(n * host.element_size()),
                                  C.c_int(2))
        if rc != 0:
            raise CanopyError(_capi.CF_ERR_CUDA, f"cudaMemcpy device->host failed with {rc}")
        return host

    def scalars(self):
        c = self.c
        return {
            "amax": self._read(c.amax).item(), "scale": self._read(c.scale).item(),
            "descale": self._read(c.descale).item(), "scale_snapshot": self._read(c.scale_snapshot).item(),
            "descale_snapshot": self._read(c.descale_snapshot).item(),
            "history": self._read(c.history, n=8).tolist(),
            "cursor": self._read(c.history_cursor, torch.int32).item(),
            "count": self._read(c.history_count, torch.int32).item(),
            "fp8_max": c.fp8_max, "init": c.init, "calib_remaining": c.calib_remaining,
        }


class Fp8Weight:
    """One FP8-cached weight (Fp8Slot, src/trainer.cu:3284-3294): bf16 master plus both E4M3 layouts."""

    def __init__(self, w, stored_out_major):
        assert w.dtype == torch.bfloat16 and w.dim() == 2 and w.is_contiguous()
        self.w = w
        if stored_out_major:
            self.out_dim, self.in_dim = w.shape
        else:
            self.in_dim, self.out_dim = w.shape
        self.fwd8 = torch.empty(self.out_dim, self.in_dim, dtype=torch.uint8, device=w.device)
        self.bwd8 = torch.empty(self.in_dim, self.out_dim, dtype=torch.uint8, device=w.device)
        self.scalars = torch.zeros(12, dtype=torch.float32, device=w.device)   # 16-byte aligned amax/scale/descale
        self.amax, self.scale, self.descale = self.scalars[0:1], self.scalars[4:5], self.scalars[8:9]
        self.c = _capi.Fp8WeightStruct(w.data_ptr(), self.fwd8.data_ptr(), self.bwd8.data_ptr(), self.amax.data_ptr(),
                                       self.scale.data_ptr(), self.descale.data_ptr(), self.in_dim, self.out_dim,
                                       int(stored_out_major))


def refresh_fp8_weight(weight, recompute_amax=True):
    check(_L().cf_refresh_fp8_weight(C.byref(weight.c), int(recompute_amax), _s()))


def fp8_quant_act(ctx, slot, x, out8=None, is_recompute=False, n=None):
    dst = C.c_void_p(ctx.act8_ptr()) if out8 is None else _p(out8)
    check(_L().cf_fp8_quant_act(ctx.handle, C.byref(slot.c), _p(x), x.numel() if n is None else n, dst, _s(),
                                int(is_recompute)))


def fp8_swiglu_quant_act(ctx, slot, gate, up, ld_in, rows, cols, out8):
    check(_L().cf_fp8_swiglu_quant_act(ctx.handle, C.byref(slot.c), _p(gate), _p(up), ld_in, rows, cols, _p(out8), _s()))


def fp8_interleave_gate_up(w_gateup8):
    """[E, 2F, K] with gate rows first -> the 32-row interleaved layout the fused SwiGLU GEMM reads."""
    E, F2, K = w_gateup8.shape
    F = F2 // 2
    out = torch.empty_like(w_gateup8)
    gate = w_gateup8[:, :F].contiguous()
    up = w_gateup8[:, F:].contiguous()
    check(_L().cf_fp8_interleave_gate_up(_p(gate), _p(up), _p(out), E, F, K, _s()))
    return out


def gemm_fp8_swiglu_quant_act(ctx, slot, num_segments, num_weights, segment_weight, max_total_rows, F, K, counts, offsets, A,
                              lda, a_is_e5m2, a_descale, per_segment_a_descale, w_interleaved, w_descale, h8, ldh):
    check(_L().cf_gemm_fp8_swiglu_quant_act(ctx.handle, C.byref(slot.c), num_segments, num_weights, _p(segment_weight),
                                            max_total_rows, F, K, _p(counts), _p(offsets), _p(A), lda, int(a_is_e5m2),
                                            _p(a_descale), int(per_segment_a_descale), _p(w_interleaved), _p(w_descale),
                                            _p(h8), ldh, _s()))


# ---------------------------------------------------------------- GEMMs
def _epi(bias, bias_mode, a_row_descale, b_col_descale, out_fp32=False):
    if bias is None and a_row_descale is None and b_col_descale is None and not out_fp32:
        return None
    return C.byref(_capi.GemmEpilogue(bias.data_ptr() if bias is not None else None, bias_mode,
                                      a_row_descale.data_ptr() if a_row_descale is not None else None,
                                      b_col_descale.data_ptr() if b_col_descale is not None else None, int(out_fp32)))


def lt_gemm_fp8_nt(ctx, M, N, K, A, lda, a_is_e5m2, a_descale, B, b_descale, Cout, ldc, bias=None, bias_mode=0,
                   a_row_descale=None, b_col_descale=None):
    """C[M,N] = (dA*dB) * A8[M,K] . B8[N,K]^T  (src/trainer.cu:4498-4534). C is bf16 like the reference's output;
    a float32 C selects the fp32 partial-product form used by row-parallel (K-sharded) GEMMs."""
    out_fp32 = Cout.dtype == torch.float32
    check(_L().cf_gemm_fp8_nt(ctx.handle, M, N, K, _p(A), lda, int(a_is_e5m2), _p(a_descale), _p(B), _p(b_descale),
                              _p(Cout), ldc, _epi(bias, bias_mode, a_row_descale, b_col_descale, out_fp32), _s()))


def lt_gemm_fp8_tn_accum_f32(ctx, M, N, K, Xt, ds_x, dYt, ds_dy, dW, ldc):
    """dW[M,N] += (dsx*dsdy) * Xt[M,K] . dYt[N,K]^T; dW fp32 or bf16 (src/trainer.cu:4596-4691)."""
    fn = _L().cf_gemm_fp8_tn_accum_f32 if dW.dtype == torch.float32 else _L().cf_gemm_fp8_tn_accum_bf16
    check(fn(ctx.handle, M, N, K, _p(Xt), _p(ds_x), _p(dYt), _p(ds_dy), _p(dW), ldc, _s()))


def gemm_fp8_dw_accum(ctx, M, N, K, X8, ldx, ds_x, dY8, ldy, ds_dy, dW, ldc):
    """dW[M,N] += X8[K,M]^T . dY8[K,N] straight from the un-transposed operands (fp32 or bf16 dW)."""
    fn = _L().cf_gemm_fp8_dw_accum_f32 if dW.dtype == torch.float32 else _L().cf_gemm_fp8_dw_accum_bf16
    check(fn(ctx.handle, M, N, K, _p(X8), ldx, _p(ds_x), _p(dY8), ldy, _p(ds_dy), _p(dW), ldc, _s()))


def gemm_fp8_nt_reduce_scatter(ctx, M, N, K_local, A, lda, a_is_e5m2, a_descale, B, b_descale, slice_ptrs,
                               a_row_descale=None, b_col_descale=None):
    """Row-parallel GEMM whose epilogue adds every row slice of the fp32 product into its owner's accumulation slice
    (slice_ptrs: device addresses, one per rank, as mapped in this process)."""
    arr = (C.c_void_p * len(slice_ptrs))(*[C.c_void_p(int(x)) for x in slice_ptrs])
    check(_L().cf_gemm_fp8_nt_reduce_scatter_f32(ctx.handle, M, N, K_local, _p(A), lda, int(a_is_e5m2), _p(a_descale), _p(B),
                                                 _p(b_descale), _p(a_row_descale), _p(b_col_descale), arr, len(slice_ptrs), _s()))


def f32_to_bf16_and_zero(acc, out):
    check(_L().cf_f32_to_bf16_and_zero(_p(acc), _p(out), acc.numel(), _s()))


def gemm_fp8_nn(ctx, M, N, K, A, lda, a_is_e5m2, a_descale, B_kn, ldb, b_descale, Cout, ldc, accumulate=False):
    """C[M,N] = A[M,K] . B[K,N]: the dgrad direction, reading the forward weight cache ([out,in] = [K,N]) as it lies."""
    check(_L().cf_gemm_fp8_nn(ctx.handle, M, N, K, _p(A), lda, int(a_is_e5m2), _p(a_descale), _p(B_kn), ldb, _p(b_descale),
                              _p(Cout), ldc, int(accumulate), _s()))


def gemm_fp8_nn_grouped(ctx, num_groups, max_total_rows, N, K, counts, offsets, A, lda, a_is_e5m2, a_descale, B_stacked_kn,
                        b_descale, Cout, ldc, accumulate=False):
    """Ragged per-expert dgrad over the stacked forward cache [E, K, N] (no transposed cache)."""
    check(_L().cf_gemm_fp8_nn_grouped(ctx.handle, num_groups, max_total_rows, N, K, _p(counts), _p(offsets), _p(A), lda,
                                      int(a_is_e5m2), _p(a_descale), _p(B_stacked_kn), _p(b_descale), _p(Cout), ldc,
                                      int(accumulate), _s()))


def gemm_fp8_nt_grouped(ctx, num_experts, max_total_rows, N, K, counts, offsets, A, lda, a_is_e5m2, a_descale,
                        per_expert_a_descale, B, b_descale, Cout, ldc):
    check(_L().cf_gemm_fp8_nt_grouped(ctx.handle, num_experts, max_total_rows, N, K, _p(counts), _p(offsets), _p(A),
                                      lda, int(a_is_e5m2), _p(a_descale), int(per_expert_a_descale), _p(B),
                                      _p(b_descale), _p(Cout), ldc, _s()))


def gemm_fp8_nt_segments(ctx, num_segments, num_weights, segment_weight, max_total_rows, N, K, counts, offsets, A, lda,
                         a_is_e5m2, a_descale, per_segment_a_descale, B, b_descale, Cout, ldc):
    check(_L().cf_gemm_fp8_nt_segments(ctx.handle, num_segments, num_weights, _p(segment_weight), max_total_rows, N, K,
                                       _p(counts), _p(offsets), _p(A), lda, int(a_is_e5m2), _p(a_descale),
                                       int(per_segment_a_descale), _p(B), _p(b_descale), _p(Cout), ldc, _s()))


def gemm_fp8_nt_segments_scatter(ctx, num_segments, num_weights, segment_weight, max_total_rows, N, K, counts, offsets, A,
                                 lda, a_is_e5m2, a_descale, per_segment_a_descale, B, b_descale, segment_out,
                                 segment_out_row0, ldc):
    """segment_out: int64 device tensor of output base addresses; segment_out_row0: int64 device tensor of first rows."""
    check(_L().cf_gemm_fp8_nt_segments_scatter(ctx.handle, num_segments, num_weights, _p(segment_weight), max_total_rows, N,
                                               K, _p(counts), _p(offsets), _p(A), lda, int(a_is_e5m2), _p(a_descale),
                                               int(per_segment_a_descale), _p(B), _p(b_descale), None, _p(segment_out),
                                               _p(segment_out_row0), ldc, _s()))


def fp8_linear_forward(ctx, slot, x, w8, w_descale, y, bias=None, bias_mode=2):
    M, K = x.shape
    N = w8.shape[0]
    check(_L().cf_fp8_linear_forward(ctx.handle, C.byref(slot.c), _p(x), M, K, _p(w8), _p(w_descale), N, _p(bias),
                                     bias_mode if bias is not None else 0, _p(y), y.stride(0), _s()))


# ---------------------------------------------------------------- elementwise + MoE
def bias_add_strided_bf16(inout, bias, rows, cols, row_stride, base):
    check(_L().cf_bias_add_strided_bf16(_p(inout), _p(bias), rows, cols, row_stride, base, _s()))


def swiglu_forward(gate, up, out, n=None):
    check(_L().cf_swiglu_forward(_p(gate), _p(up), _p(out), gate.numel() if n is None else n, _s()))


def lion_step(w, m, grad, lr, beta1, beta2, wd, weight_amax=None, sr_seed=0):
    """lion_step (include/ida_native/kernels.hpp:1089-1108); m float32 or bfloat16 selects the overload."""
    fn = _L().cf_lion_step_f32_state if m.dtype == torch.float32 else _L().cf_lion_step_bf16_state
    check(fn(_p(w), _p(m), _p(grad), w.numel(), lr, beta1, beta2, wd, _s(), _p(weight_amax), sr_seed))


def lion_step_quantize(w, m, grad, lr, beta1, beta2, wd, weight_amax, quant_amax, scale_out, descale_out, w8,
                       w8_transposed=None, sr_seed=0):
    """lion_step that also writes the E4M3 cache(s) of the [rows, cols] weight in the same pass (scale from quant_amax,
    the amax an earlier step left; this step's amax goes to weight_amax)."""
    rows, cols = w.shape
    fn = _L().cf_lion_step_f32_state_quantize if m.dtype == torch.float32 else _L().cf_lion_step_bf16_state_quantize
    check(fn(_p(w), _p(m), _p(grad), rows, cols, lr, beta1, beta2, wd, _s(), _p(weight_amax), sr_seed, _p(quant_amax),
             _p(scale_out), _p(descale_out), _p(w8), _p(w8_transposed)))


def gelu_forward(x, out):
    check(_L().cf_gelu_forward(_p(x), _p(out), x.numel(), _s()))


def fp8_quantize_rowwise_e4m3(x, out, row_descale, row_scale=None, rows=None, cols=None, ld_x=None, ld_out=None):
    rows = x.shape[0] if rows is None else rows
    cols = x.shape[1] if cols is None else cols
    check(_L().cf_fp8_quantize_rowwise_e4m3(_p(x), x.stride(0) if ld_x is None else ld_x, _p(out),
                                            out.stride(0) if ld_out is None else ld_out, _p(row_scale), _p(row_descale),
                                            rows, cols, _s()))


def fp8_quantize_rowwise_given_amax_e4m3(x, out, row_amax, row_descale, row_scale=None, rows=None, cols=None):
    rows = x.shape[0] if rows is None else rows
    cols = x.shape[1] if cols is None else cols
    check(_L().cf_fp8_quantize_rowwise_given_amax_e4m3(_p(x), x.stride(0), _p(out), out.stride(0), _p(row_amax),
                                                       _p(row_scale), _p(row_descale), rows, cols, _s()))


def gemm_fp8_swiglu_bf16_rowamax(ctx, M, F, K, A, lda, a_is_e5m2, a_descale, a_row_descale, w_interleaved, w_descale,
                                 w_col_descale_interleaved, h, row_amax):
    """Gate/up GEMM + SwiGLU in one launch: h bf16 [M, F] and max|h| per row (row_amax, zeroed by the caller)."""
    check(_L().cf_gemm_fp8_swiglu_bf16_rowamax(ctx.handle, M, F, K, _p(A), lda, int(a_is_e5m2), _p(a_descale),
                                               _p(a_row_descale), _p(w_interleaved), _p(w_descale),
                                               _p(w_col_descale_interleaved), _p(h), h.stride(0), _p(row_amax), _s()))


def interleave_gate_up_vector(v, F):
    """A per-output-row vector of the [2F, K] gate/up weight (gate rows first) in the 32-row interleaved order of
    fp8_interleave_gate_up: [g0..g31, u0..u31, g32..g63, u32..u63, ...]."""
    g, u = v[:F].reshape(F // 32, 32), v[F:].reshape(F // 32, 32)
    return torch.stack([g, u], dim=1).reshape(2 * F).contiguous()


def swiglu_quantize_rowwise_e4m3(gate, up, out, row_descale, rows, cols, ld_in, ld_out=None, row_scale=None):
    check(_L().cf_swiglu_quantize_rowwise_e4m3(_p(gate), _p(up), ld_in, _p(out), cols if ld_out is None else ld_out,
                                               _p(row_scale), _p(row_descale), rows, cols, _s()))


def rmsnorm_forward(x, scale, out, rms, rows, H, eps=1e-6):
    """out = bf16(x / rms * scale) per row, rms kept for the backward pass (kernels/rmsnorm.cu:101-108)."""
    check(_L().cf_rmsnorm_forward(_p(x), _p(scale), _p(out), _p(rms), rows, H, eps, _s()))


def rmsnorm_quantize_e4m3_record(x, scale, normed, rms, out8, quant_scale, amax, rows, H, eps=1e-6):
    """rmsnorm_forward + fp8_quantize_e4m3_record in one pass; normed / rms may be None."""
    check(_L().cf_rmsnorm_quantize_e4m3_record(_p(x), _p(scale), _p(normed), _p(rms), _p(out8), _p(quant_scale), _p(amax),
                                               rows, H, eps, _s()))


def rmsnorm_quantize_rowwise_e4m3(x, scale, normed, rms, out8, row_descale, rows, H, eps=1e-6, row_scale=None):
    check(_L().cf_rmsnorm_quantize_rowwise_e4m3(_p(x), _p(scale), _p(normed), _p(rms), _p(out8), _p(row_scale),
                                                _p(row_descale), rows, H, eps, _s()))


def fp8_rmsnorm_quant_act(ctx, slot, x, scale, normed, rms, rows, H, out8, eps=1e-6):
    """rmsnorm_forward followed by fp8_quant_act on its output (src/trainer.cu:6097,6115) as one pass."""
    check(_L().cf_fp8_rmsnorm_quant_act(ctx.handle, C.byref(slot.c), _p(x), _p(scale), _p(normed), _p(rms), rows, H, eps,
                                        _p(out8), _s()))


def rmsnorm_clip_forward(x, scale, out, rms, rows, H, clip_ceiling, eps=1e-6):
    """rmsnorm_forward followed by act_row_clip (fixed ceiling) in one pass."""
    check(_L().cf_rmsnorm_clip_forward(_p(x), _p(scale), _p(out), _p(rms), rows, H, eps, clip_ceiling, _s()))


def rmsnorm_clip_quantize_e4m3_record(x, scale, normed, rms, out8, quant_scale, amax, rows, H, clip_ceiling, eps=1e-6):
    check(_L().cf_rmsnorm_clip_quantize_e4m3_record(_p(x), _p(scale), _p(normed), _p(rms), _p(out8), _p(quant_scale),
                                                    _p(amax), rows, H, eps, clip_ceiling, _s()))


def fp8_rmsnorm_clip_quant_act(ctx, slot, x, scale, normed, rms, rows, H, out8, clip_ceiling, eps=1e-6):
    """rmsnorm_forward, act_row_clip and fp8_quant_act (src/trainer.cu:6097-6115) as one pass."""
    check(_L().cf_fp8_rmsnorm_clip_quant_act(ctx.handle, C.byref(slot.c), _p(x), _p(scale), _p(normed), _p(rms), rows, H, eps,
                                             clip_ceiling, _p(out8), _s()))


def swiglu_quantize_e4m3_record(gate, up, out, scale, amax, rows, cols, ld_in, ld_out=None):
    check(_L().cf_swiglu_quantize_e4m3_record(_p(gate), _p(up), ld_in, _p(out), cols if ld_out is None else ld_out,
                                              _p(scale), _p(amax), rows, cols, _s()))


def moe_topk_route_f32(scores, rows, num_experts, top_k, row_sum_save=None, scores_save=None, normalize_topk=True):
    check(_L().cf_moe_topk_route_f32(_p(scores), rows, num_experts, top_k, _s(), _p(row_sum_save), _p(scores_save),
                                     int(normalize_topk)))


def moe_build_expert_row_lists(route_weights, counts, row_indices, rows, num_experts):
    check(_L().cf_moe_build_expert_row_lists(_p(route_weights), _p(counts), _p(row_indices), rows, num_experts, _s()))


def moe_expert_offsets_from_counts(counts, offsets, num_experts):
    check(_L().cf_moe_expert_offsets_from_counts(_p(counts), _p(offsets), num_experts, _s()))


def moe_gather_rows_u8(src, dst, row_indices, n_rows, width):
    check(_L().cf_moe_gather_rows_u8(_p(src), _p(dst), _p(row_indices), n_rows, width, _s()))


def moe_gather_rows_bf16(src, dst, row_indices, n_rows, width):
    check(_L().cf_moe_gather_rows_bf16(_p(src), _p(dst), _p(row_indices), n_rows, width, _s()))


def moe_scatter_accumulate_rows_bf16(mixed, compact, route_weights, row_indices, n_rows, expert_idx, num_experts, H):
    check(_L().cf_moe_scatter_accumulate_rows_bf16(_p(mixed), _p(compact), _p(route_weights), _p(row_indices), n_rows,
                                                   expert_idx, num_experts, H, _s()))


def moe_scale_accumulate_bf16(mixed, term, route_weights, rows, expert_idx, num_experts, H):
    check(_L().cf_moe_scale_accumulate_bf16(_p(mixed), _p(term), _p(route_weights), rows, expert_idx, num_experts, H, _s()))


def moe_gather_all_u8(src, dst, row_indices, counts, offsets, rows, num_experts, width):
    check(_L().cf_moe_gather_all_u8(_p(src), _p(dst), _p(row_indices), _p(counts), _p(offsets), rows, num_experts, width, _s()))


def moe_combine_all_bf16(mixed, compact, route_weights, row_indices, counts, offsets, rows, num_experts, H):
    check(_L().cf_moe_combine_all_bf16(_p(mixed), _p(compact), _p(route_weights), _p(row_indices), _p(counts),
                                       _p(offsets), rows, num_experts, H, _s()))


def moe_combine_sorted_bf16(mixed, compact, route_weights, row_indices, counts, offsets, rows, num_experts, H,
                            accumulate=True):
    """One pass over the token rows (ascending dispatch lists): mixed is read (accumulate) or started from zero, and
    written once; equals zero-fill + moe_combine_all_bf16 bit for bit."""
    check(_L().cf_moe_combine_sorted_bf16(_p(mixed), _p(compact), _p(route_weights), _p(row_indices), _p(counts),
                                          _p(offsets), rows, num_experts, H, int(accumulate), _s()))


def moe_expand_route_replicas(route_weights, replica_weights, rows, num_experts, num_replicas, replica_start,
                              replica_cum_share, first_row=0):
    """[rows, E] sparse route weights -> [rows, V] over expert replicas (one replica per selected expert and row)."""
    check(_L().cf_moe_expand_route_replicas(_p(route_weights), _p(replica_weights), rows, num_experts, num_replicas,
                                            _p(replica_start), _p(replica_cum_share), int(first_row) & 0xffffffff, _s()))


def moe_route_dispatch_scratch_ints(rows, num_lists):
    return int(_L().cf_moe_route_dispatch_scratch_ints(rows, num_lists))


def moe_route_dispatch_lists(scores, rows, num_experts, top_k, counts, offsets, row_indices, scratch, normalize=True,
                             replica_weights=None, num_replicas=0, replica_start=None, replica_cum_share=None, first_row=0,
                             row_sum_save=None, scores_save=None):
    """Route + (replica choice) + ascending dispatch lists + counts + offsets in one call: the outputs of
    moe_topk_route_f32, [moe_expand_route_replicas,] moe_build_expert_row_lists and moe_expert_offsets_from_counts."""
    check(_L().cf_moe_route_dispatch_lists(_p(scores), rows, num_experts, top_k, int(normalize), _p(row_sum_save),
                                           _p(scores_save), _p(replica_weights), num_replicas, _p(replica_start),
                                           _p(replica_cum_share), int(first_row) & 0xffffffff, _p(counts), _p(offsets),
                                           _p(row_indices), _p(scratch), scratch.numel(), _s()))


def peer_barrier(ctx, flag_arrays, world, rank, epoch, limit_ms=2000):
    """Barrier between the ranks of one box done by the GPUs (flag words in peer-mapped memory); flag_arrays: int64
    device tensor of the ranks' flag-array addresses as mapped in this process."""
    check(_L().cf_peer_barrier(ctx.handle, _p(flag_arrays), world, rank, int(epoch) & 0xffffffff, int(limit_ms), _s()))


def peer_share_i32(ctx, src, n, tables, flag_arrays, world, rank, epoch, limit_ms=2000):
    """This rank's n int32 words into row `rank` of every rank's [world, n] table, then the flag-word barrier, in one
    launch (tables / flag_arrays: int64 device tensors of addresses as mapped in this process)."""
    check(_L().cf_peer_share_i32(ctx.handle, _p(src), int(n), _p(tables), _p(flag_arrays), world, rank,
                                 int(epoch) & 0xffffffff, int(limit_ms), _s()))


ROW_RUN_BYTES = 24      # sizeof(cf_row_run): two int64 and two int32


def moe_ep_plan(counts_all, world, rank, num_replicas, range_lo, range_hi, send_runs, group_counts, group_offsets,
                return_runs, recv_capacity_rows=0, ctx=None):
    """Device-side plan of one expert-parallel layer from the gathered count table (no host copy)."""
    check(_L().cf_moe_ep_plan(_p(counts_all), world, rank, num_replicas, _p(range_lo), _p(range_hi), _p(send_runs),
                              _p(group_counts), _p(group_offsets), _p(return_runs), int(recv_capacity_rows),
                              ctx.handle if ctx is not None else None, _s()))


def moe_send_row_runs(src, row_indices, index_stride, runs, num_runs, max_rows_per_run, dst_bases, row_bytes,
                      num_dst, dst_rows, tag_value=None, tag_bases=None, ctx=None):
    """Copies planned runs of rows into (peer) destination buffers; optional gather through an index table and a
    per-row float tag. dst_bases / tag_bases: int64 device tensors of num_dst base addresses of dst_rows rows each; a
    run that leaves its destination is skipped and reported through ctx.poll_status()."""
    check(_L().cf_moe_send_row_runs(_p(src), _p(row_indices), index_stride, _p(runs), num_runs, max_rows_per_run,
                                    _p(dst_bases), row_bytes, _p(tag_value), _p(tag_bases), int(num_dst), int(dst_rows),
                                    ctx.handle if ctx is not None else None, _s()))


def gemm_fp8_nt_grouped_return(ctx, num_groups, max_total_rows, N, K, counts, offsets, A, lda, a_is_e5m2, a_descale, B,
                               b_descale, return_runs, runs_per_group, dst_ptrs, dst_rows, ldc):
    """Ragged grouped GEMM whose epilogue stores every run of rows into its destination buffer (dst_ptrs: device
    addresses as mapped in this process, one per rank)."""
    arr = (C.c_void_p * len(dst_ptrs))(*[C.c_void_p(int(x)) for x in dst_ptrs])
    check(_L().cf_gemm_fp8_nt_grouped_return(ctx.handle, num_groups, max_total_rows, N, K, _p(counts), _p(offsets), _p(A),
                                             lda, int(a_is_e5m2), _p(a_descale), _p(B), _p(b_descale), _p(return_runs),
                                             runs_per_group, arr, len(dst_ptrs), dst_rows, ldc, _s()))


def moe_grouped_expert_forward_fp8(ctx, hidden, fcin_descale, fcin_is_e5m2, route_weights, counts, offsets, row_indices,
                                   fc_in_w, fc_in_descale, fc_out_w, fc_out_descale, mixed, rows, H, Ie, num_experts,
                                   total_selected_rows):
    check(_L().cf_moe_grouped_expert_forward_fp8(ctx.handle, _p(hidden), _p(fcin_descale), int(fcin_is_e5m2),
                                                 _p(route_weights), _p(counts), _p(offsets), _p(row_indices),
                                                 _p(fc_in_w), _p(fc_in_descale), _p(fc_out_w), _p(fc_out_descale),
                                                 _p(mixed), rows, H, Ie, num_experts, total_selected_rows, _s()))


# ---------------------------------------------------------------- block-scaled FP8 (one scale per 128 values)
BLOCK = 128
_bf16, _u8, _f32, _i32 = torch.bfloat16, torch.uint8, torch.float32, torch.int32


def _refuse(what):
    """A call whose tensors do not fit together is refused before any pointer reaches the library."""
    raise CanopyError(_capi.CF_ERR_INVALID_ARG, what)


_INT_MAX = 0x7fffffff              # of a C int: ctypes would cut a larger size down without a word


def _blocks(n):
    return (n + 127) >> 7


def _on(*tensors):
    """Every tensor is on the current device, whose stream the call goes to."""
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _refuse(f"tensors on the current device (cuda:{dev}) expected, got one on {t.device}")


def _a(t):
    """Address of a tensor (an integer: ctypes takes it as it is, a small call spends its time here)."""
    return None if t is None else t.data_ptr()


def _mat(t, dtype, rows, cols, what):
    """Row pitch of a [rows, cols] matrix with contiguous columns and rows that do not overlap."""
    if t.dtype is not dtype or t.shape != (rows, cols):
        _refuse(f"{what}: {dtype} [{rows}, {cols}] expected, got {t.dtype} {tuple(t.shape)}")
    ld, step = t.stride()
    if (step != 1 and cols > 1) or (ld < cols and rows > 1):
        _refuse(f"{what}: columns must be contiguous and rows must not overlap")
    if rows > _INT_MAX or cols > _INT_MAX or (ld > _INT_MAX and rows > 1):
        _refuse(f"{what}: sizes and pitches go up to 2^31 - 1")
    return ld if rows > 1 else (cols + 15) & ~15       # the pitch of a single row addresses no memory


def _scales(t, rows, cols, what):
    """Strides of a matrix of descales (any)."""
    if t.dtype is not _f32 or t.shape != (rows, cols):
        _refuse(f"{what}: float32 [{rows}, {cols}] expected, got {t.dtype} {tuple(t.shape)}")
    return t.stride()


def _dense(t, dtype, shape, what):
    if t is not None and (t.dtype is not dtype or t.shape != shape or not t.is_contiguous()):
        _refuse(f"{what}: contiguous {dtype} {list(shape)} expected, got {t.dtype} {tuple(t.shape)}")
    if len(shape) == 2 and max(shape) > _INT_MAX:
        _refuse(f"{what}: sizes go up to 2^31 - 1")


def block128_row_descale(rows, cols, device="cuda"):
    """Descales of row groups, [rows, ceil(cols / 128)], the rows next to each other in memory (what the GEMM reads best)."""
    return torch.empty((_blocks(cols), rows), dtype=torch.float32, device=device).t()


def _group_outputs(rows, cols, row8, row_descale, col8, col_descale):
    if (row8 is None) != (row_descale is None) or (col8 is None) != (col_descale is None):
        _refuse("codes and descales go together")
    if row8 is None and col8 is None:
        _refuse("no output")
    r = c = (None, 0, None, 0, 0)
    if row8 is not None:
        r = (_a(row8), _mat(row8, _u8, rows, cols, "row8"), _a(row_descale), *_scales(row_descale, rows, _blocks(cols), "row_descale"))
    if col8 is not None:
        c = (_a(col8), _mat(col8, _u8, rows, cols, "col8"), _a(col_descale), *_scales(col_descale, _blocks(rows), cols, "col_descale"))
    return r + c


def fp8_quantize_block128(x, row8=None, row_descale=None, col8=None, col_descale=None, is_e5m2=False):
    """Codes of a bf16 matrix with one scale per 128 values of a row (row8, row_descale [rows, ceil(cols/128)]) and / or per
    128 values of a column (col8, col_descale [ceil(rows/128), cols]), from one read."""
    _on(x, row8, row_descale, col8, col_descale)
    rows, cols = x.shape
    check(_L().cf_fp8_quantize_block128(_a(x), _mat(x, _bf16, rows, cols, "x"), rows, cols, is_e5m2,
                                        *_group_outputs(rows, cols, row8, row_descale, col8, col_descale), _s()))


def swiglu_quantize_block128(gate, up, row8=None, row_descale=None, col8=None, col_descale=None):
    """fp8_quantize_block128 of silu(gate) * up (E4M3, no bf16 rounding in between); gate and up share a row pitch."""
    _on(gate, up, row8, row_descale, col8, col_descale)
    rows, cols = gate.shape
    ld = _mat(gate, _bf16, rows, cols, "gate")
    if _mat(up, _bf16, rows, cols, "up") != ld:
        _refuse("gate and up must have the same row pitch")
    check(_L().cf_swiglu_quantize_block128(_a(gate), _a(up), ld, rows, cols,
                                           *_group_outputs(rows, cols, row8, row_descale, col8, col_descale), _s()))


def swiglu_backward_quantize_block128(gate, up, dh, row8=None, row_descale=None, col8=None, col_descale=None, is_e5m2=False):
    """Codes of the gradient of silu(gate) * up: [rows, 2 cols], d gate first, d up behind it; cols a multiple of 128."""
    _on(gate, up, dh, row8, row_descale, col8, col_descale)
    rows, cols = gate.shape
    ld = _mat(gate, _bf16, rows, cols, "gate")
    if _mat(up, _bf16, rows, cols, "up") != ld:
        _refuse("gate and up must have the same row pitch")
    check(_L().cf_swiglu_backward_quantize_block128(_a(gate), _a(up), ld, _a(dh), _mat(dh, _bf16, rows, cols, "dh"), rows, cols, is_e5m2,
                                                    *_group_outputs(rows, 2 * cols, row8, row_descale, col8, col_descale), _s()))


def fp8_quantize_block128x128(w, w8, descale):
    """E4M3 codes of a weight [rows, cols], or of a stack [n, rows, cols], with one scale per 128x128 block
    (descale [..., ceil(rows/128), ceil(cols/128)])."""
    _on(w, w8, descale)
    if w.dim() not in (2, 3) or w8.shape != w.shape or descale.dim() != w.dim():
        _refuse("weight, codes and descales: shapes differ")
    n = w.shape[0] if w.dim() == 3 else 1
    if n > _INT_MAX:
        _refuse("a stack of more than 2^31 - 1 weights")
    rows, cols = w.shape[-2:]
    if n == 0 or rows == 0 or cols == 0:
        return
    stacked = w.dim() == 3
    if descale.dtype is not _f32 or descale.shape != (*w.shape[:-2], _blocks(rows), _blocks(cols)) or \
            (descale.stride(-1) != 1 and descale.shape[-1] > 1):
        _refuse("descale: float32 with contiguous rows of blocks expected")
    w0, q0, d0 = (w[0], w8[0], descale[0]) if stacked else (w, w8, descale)
    ld_d = d0.stride(0) if d0.shape[0] > 1 else max(d0.stride(0), d0.shape[1])
    check(_L().cf_fp8_quantize_block128x128(_a(w), _mat(w0, _bf16, rows, cols, "w"), w.stride(0) if stacked else 0, n, rows, cols, _a(w8),
                                            _mat(q0, _u8, rows, cols, "w8"), w8.stride(0) if stacked else 0, _a(descale), ld_d,
                                            descale.stride(0) if stacked else 0, _s()))


def add_rmsnorm_quantize_block128(x, residual, scale, h, rms=None, normed=None, out8=None, descale=None, eps=1e-6):
    """h = bf16(x + residual), RMS norm of h with gain `scale`, codes and row-group descales of the normalised row (and / or
    its bf16 copy `normed`), in one pass. residual may be None (then h may be, too); h may be x or residual itself."""
    _on(x, residual, scale, h, rms, normed, out8, descale)
    shape = rows, H = x.shape
    _dense(x, _bf16, shape, "x")
    _dense(residual, _bf16, shape, "residual")
    _dense(h, _bf16, shape, "h")
    _dense(normed, _bf16, shape, "normed")
    _dense(scale, _bf16, (H,), "scale")
    _dense(rms, _f32, (rows,), "rms")
    if (out8 is None) != (descale is None):
        _refuse("codes and descales go together")
    o = (None, 0, None, 0, 0)
    if out8 is not None:
        o = (_a(out8), _mat(out8, _u8, rows, H, "out8"), _a(descale), *_scales(descale, rows, _blocks(H), "descale"))
    check(_L().cf_add_rmsnorm_quantize_block128(_a(x), _a(residual), _a(scale), _a(h), _a(normed), _a(rms), *o, rows, H, eps, _s()))


def add_rmsnorm_backward_scratch_floats(rows, H):
    return int(_L().cf_add_rmsnorm_backward_scratch_floats(rows, H))


def add_rmsnorm_backward(dy, h, scale, rms, dh, dx, dscale=None, scratch=None, accumulate_dscale=False):
    """Gradient of the residual addition + RMS norm: dx (of x and of the residual alike) from dy and the gradient dh of the
    residual stream (or None); dscale float32 [H], stored or added to, or None. dx may be dy or dh itself."""
    _on(dy, h, scale, rms, dh, dx, dscale, scratch)
    shape = rows, H = h.shape
    _dense(h, _bf16, shape, "h")
    _dense(dy, _bf16, shape, "dy")
    _dense(dh, _bf16, shape, "dh")
    _dense(dx, _bf16, shape, "dx")
    _dense(scale, _bf16, (H,), "scale")
    _dense(rms, _f32, (rows,), "rms")
    _dense(dscale, _f32, (H,), "dscale")
    floats = 0
    if scratch is not None:
        floats = scratch.numel()
        _dense(scratch, _f32, (floats,), "scratch")
    check(_L().cf_add_rmsnorm_backward(_a(dy), _a(h), _a(scale), _a(rms), _a(dh), _a(dx), _a(dscale), accumulate_dscale, _a(scratch),
                                       floats, rows, H, _s()))


def _output(out, M, N):
    f32 = out.dtype is _f32
    return _a(out), _mat(out, _f32 if f32 else _bf16, M, N, "out"), f32


def gemm_fp8_block128_nt(ctx, A8, a_descale, B8, b_descale, out, a_is_e5m2=False, accumulate=False):
    """out[M,N] (bf16 or float32) = A8[M,K] . B8[N,K]^T with a_descale [M, ceil(K/128)] and b_descale [ceil(N/128), ceil(K/128)]
    (128x128 blocks, weights) or [N, ceil(K/128)] (row groups; taken for blocks where the two shapes are the same, N = 1)."""
    _on(A8, a_descale, B8, b_descale, out)
    (M, K), N = A8.shape, B8.shape[0]
    nb, kb = _blocks(N), _blocks(K)
    per = BLOCK if b_descale.shape[0] == nb else 1
    check(_L().cf_gemm_fp8_block128_nt(ctx.handle, M, N, K, _a(A8), _mat(A8, _u8, M, K, "A8"), a_is_e5m2, _a(a_descale),
                                       *_scales(a_descale, M, kb, "a_descale"), _a(B8), _mat(B8, _u8, N, K, "B8"), _a(b_descale),
                                       *_scales(b_descale, nb if per == BLOCK else N, kb, "b_descale"), per, *_output(out, M, N),
                                       accumulate, _s()))


def gemm_fp8_block128_nt_grouped(ctx, counts, offsets, A8, a_descale, B8, b_descale, out, a_is_e5m2=False):
    """Rows [offsets[e], +counts[e]) of the compact A8 times expert e of the stacked B8 [E, N, K] (b_descale
    [E, ceil(N/128), ceil(K/128)]) into the same rows of the bf16 out; the other rows are left as they are."""
    _on(counts, offsets, A8, a_descale, B8, b_descale, out)
    (T, K), (E, N, _) = A8.shape, B8.shape
    if not 0 < E <= _INT_MAX:
        _refuse("B8: no experts, or more than 2^31 - 1")
    _dense(counts, _i32, (E,), "counts")
    _dense(offsets, _i32, (E,), "offsets")
    ldb = _mat(B8[0], _u8, N, K, "B8")
    if E > 1:
        if N == 1:
            ldb = B8.stride(0)
            if ldb > _INT_MAX:
                _refuse("B8: pitches go up to 2^31 - 1")
        if B8.stride(0) != N * ldb:
            _refuse("B8: the experts must lie behind one another")
    if b_descale.dtype is not _f32 or b_descale.shape != (E, _blocks(N), _blocks(K)) or (b_descale.stride(2) != 1 and b_descale.shape[2] > 1):
        _refuse("b_descale: float32 [E, ceil(N/128), ceil(K/128)] expected")
    check(_L().cf_gemm_fp8_block128_nt_grouped(ctx.handle, E, T, N, K, _a(counts), _a(offsets), _a(A8), _mat(A8, _u8, T, K, "A8"), a_is_e5m2,
                                               _a(a_descale), *_scales(a_descale, T, _blocks(K), "a_descale"), _a(B8), ldb, _a(b_descale),
                                               b_descale.stride(1), b_descale.stride(0), _a(out), _mat(out, _bf16, T, N, "out"), _s()))


def gemm_fp8_block128_nn(ctx, A8, a_descale, B8_kn, b_descale, out, a_is_e5m2=False, accumulate=False):
    """Data gradient: out[M,N] = A8[M,K] . B8[K,N], the weight read from its forward cache ([out, in] = [K, N]) and block descales
    [ceil(K/128), ceil(N/128)] as they lie; A8 (the gradient) with row groups along K."""
    _on(A8, a_descale, B8_kn, b_descale, out)
    (M, K), N = A8.shape, B8_kn.shape[1]
    ld_b, step = _scales(b_descale, _blocks(K), _blocks(N), "b_descale")
    if step != 1 and N > BLOCK:
        _refuse("b_descale: rows of blocks must be contiguous")
    check(_L().cf_gemm_fp8_block128_nn(ctx.handle, M, N, K, _a(A8), _mat(A8, _u8, M, K, "A8"), a_is_e5m2, _a(a_descale),
                                       *_scales(a_descale, M, _blocks(K), "a_descale"), _a(B8_kn), _mat(B8_kn, _u8, K, N, "B8_kn"),
                                       _a(b_descale), ld_b, *_output(out, M, N), accumulate, _s()))


def gemm_fp8_block128_dw(ctx, X8, x_descale, dY8, dy_descale, dW, x_is_e5m2=False, dy_is_e5m2=False, accumulate=False):
    """Weight gradient: dW[M,N] (float32 or bf16) = X8[T,M]^T . dY8[T,N] over T tokens, both with column groups of 128 tokens
    (descales [ceil(T/128), M] and [ceil(T/128), N])."""
    _on(X8, x_descale, dY8, dy_descale, dW)
    (T, M), N = X8.shape, dY8.shape[1]
    kb = _blocks(T)
    check(_L().cf_gemm_fp8_block128_dw(ctx.handle, M, N, T, _a(X8), _mat(X8, _u8, T, M, "X8"), x_is_e5m2, _a(x_descale),
                                       *_scales(x_descale, kb, M, "x_descale"), _a(dY8), _mat(dY8, _u8, T, N, "dY8"), dy_is_e5m2,
                                       _a(dy_descale), *_scales(dy_descale, kb, N, "dy_descale"), *_output(dW, M, N), accumulate, _s()))


# ---------------------------------------------------------------- composites: SwiGLU MLP (per-token scales) and MoE SwiGLU experts
def swiglu_mlp_fp8_rowwise(ctx, x, w_gateup8, w_gateup_descale, w_down8, w_down_descale, y, work=None):
    """Llama-style SwiGLU MLP in FP8 with per-token activation scales and per-output-channel weight scales
    (the reference has per-tensor scales only, so this follows the documented generalisation
    C[m,n] = dA[m] * dW[n] * acc):
        x8, dx   = rowwise_quant(x)                      [M,H]
        gu       = x8 . w_gateup8^T  (scales dx, dWgu)   [M,2F]  gate = gu[:, :F], up = gu[:, F:]
        h8, dh   = rowwise_quant(bf16(silu(gate) * up))  [M,F]
        y        = h8 . w_down8^T    (scales dh, dWd)    [M,H]
    w_gateup8 is [2F,H] (gate rows first), w_down8 is [H,F]; descales are float[2F] / float[H]."""
    M, H = x.shape
    F2 = w_gateup8.shape[0]
    F = F2 // 2
    dev = x.device
    if work is None:
        work = {}
    x8 = work.setdefault("x8", torch.empty((M, H), dtype=torch.uint8, device=dev))
    dx = work.setdefault("dx", torch.empty(M, dtype=torch.float32, device=dev))
    gu = work.setdefault("gu", torch.empty((M, F2), dtype=torch.bfloat16, device=dev))
    h8 = work.setdefault("h8", torch.empty((M, F), dtype=torch.uint8, device=dev))
    dh = work.setdefault("dh", torch.empty(M, dtype=torch.float32, device=dev))
    one = work.setdefault("one", torch.ones(4, dtype=torch.float32, device=dev))
    fp8_quantize_rowwise_e4m3(x, x8, dx)
    lt_gemm_fp8_nt(ctx, M, F2, H, x8, H, False, one, w_gateup8, one, gu, F2, a_row_descale=dx,
                   b_col_descale=w_gateup_descale)
    swiglu_quantize_rowwise_e4m3(gu, gu.view(-1)[F:], h8, dh, M, F, F2)
    lt_gemm_fp8_nt(ctx, M, y.shape[1], F, h8, F, False, one, w_down8, one, y, y.stride(0), a_row_descale=dh,
                   b_col_descale=w_down_descale)
    return work


def swiglu_mlp_fp8_rowwise_fused(ctx, x, w_gateup8_il, w_gateup_descale_il, w_down8, w_down_descale, y, work=None,
                                 amax_allreduce=None, down=None):
    """The same MLP as swiglu_mlp_fp8_rowwise with the [M, 2F] bf16 gate/up intermediate fused away: the gate/up GEMM's
    epilogue writes h = bf16(silu(gate) * up) as bf16 [M, F] and records max|h| per row, one row-wise pass quantises h
    with that amax, the down GEMM follows. Bit-identical to the unfused composite. w_gateup8_il is the [2F, H] weight in
    the 32-row interleaved layout (fp8_interleave_gate_up) with its per-row descales interleaved the same way
    (interleave_gate_up_vector).
    Sharded use (gate/up split by output features, down by its contraction dimension): F is this rank's share,
    amax_allreduce(row_amax) max-reduces the per-row amax over the ranks before the quantiser, and down(h8, dh) replaces
    the local down GEMM (partial products that the caller sums across ranks)."""
    M, H = x.shape
    F = w_gateup8_il.shape[0] // 2
    dev = x.device
    if work is None:
        work = {}
    x8 = work.setdefault("x8", torch.empty((M, H), dtype=torch.uint8, device=dev))
    dx = work.setdefault("dx", torch.empty(M, dtype=torch.float32, device=dev))
    h = work.setdefault("h", torch.empty((M, F), dtype=torch.bfloat16, device=dev))
    h8 = work.setdefault("h8", torch.empty((M, F), dtype=torch.uint8, device=dev))
    hmax = work.setdefault("hmax", torch.empty(M, dtype=torch.float32, device=dev))
    dh = work.setdefault("dh", torch.empty(M, dtype=torch.float32, device=dev))
    one = work.setdefault("one", torch.ones(4, dtype=torch.float32, device=dev))
    fp8_quantize_rowwise_e4m3(x, x8, dx)
    hmax.zero_()
    gemm_fp8_swiglu_bf16_rowamax(ctx, M, F, H, x8, H, False, None, dx, w_gateup8_il, None, w_gateup_descale_il, h, hmax)
    if amax_allreduce is not None:
        amax_allreduce(hmax)
    fp8_quantize_rowwise_given_amax_e4m3(h, h8, hmax, dh)
    if down is not None:
        down(h8, dh)
    else:
        lt_gemm_fp8_nt(ctx, M, y.shape[1], F, h8, F, False, one, w_down8, one, y, y.stride(0), a_row_descale=dh,
                       b_col_descale=w_down_descale)
    return work


class MoeSwigluFp8:
    """Top-k routed SwiGLU experts in FP8: route -> dispatch lists -> per-tensor delayed-scale
    quantise of x -> permute -> ragged gate/up GEMM -> SwiGLU + delayed-scale re-quantise -> ragged down GEMM ->
    unpermute + weighted combine. Everything is scheduled on the device (no host copy of the counts); the
    rounding points are those of the reference's SwiGLU expert maths (src/trainer.cu:6510-6529) combined with its
    FP8 quantise / GEMM semantics. Weights: w_gateup8 [E,2F,H] and w_down8 [E,H,F] with one per-tensor descale each."""

    def __init__(self, ctx, rows, H, F, E, top_k, device="cuda", fused_swiglu=False):
        """fused_swiglu: gate/up GEMM, SwiGLU and re-quantise run as one launch (cf_gemm_fp8_swiglu_quant_act) and the
        [T, 2F] bf16 intermediate is never materialised; forward() then expects w_gateup8 in the interleaved layout."""
        self.ctx, self.rows, self.H, self.F, self.E, self.k = ctx, rows, H, F, E, top_k
        self.fused_swiglu = fused_swiglu
        T = rows * top_k
        self.T = T
        self.counts = torch.zeros(E, dtype=torch.int32, device=device)
        self.offsets = torch.zeros(E, dtype=torch.int32, device=device)
        self.idx = torch.zeros((E, rows), dtype=torch.int32, device=device)
        self.x8 = torch.empty((rows, H), dtype=torch.uint8, device=device)
        self.xc = torch.empty((T, H), dtype=torch.uint8, device=device)
        self.gu = None if fused_swiglu else torch.empty((T, 2 * F), dtype=torch.bfloat16, device=device)
        self.h8 = torch.empty((T, F), dtype=torch.uint8, device=device)
        self.yc = torch.empty((T, H), dtype=torch.bfloat16, device=device)
        self.slot_x = ActSlot(ctx, E4M3_MAX)
        self.slot_h = ActSlot(ctx, E4M3_MAX)
        self.front_scratch = torch.empty(max(1, moe_route_dispatch_scratch_ints(rows, E)), dtype=torch.int32, device=device)

    def forward(self, x, route_weights, w_gateup8, w_gateup_descale, w_down8, w_down_descale, mixed, accumulate=True):
        """route_weights: float32 [rows,E] router logits, overwritten in place by the sparse route weights.
        accumulate=False: mixed is overwritten (as if it had been zero-filled first) instead of added to."""
        rows, H, F, E, T = self.rows, self.H, self.F, self.E, self.T
        moe_route_dispatch_lists(route_weights, rows, E, self.k, self.counts, self.offsets, self.idx, self.front_scratch)
        fp8_quant_act(self.ctx, self.slot_x, x, self.x8)
        moe_gather_all_u8(self.x8, self.xc, self.idx, self.counts, self.offsets, rows, E, H)
        if self.fused_swiglu:
            gemm_fp8_swiglu_quant_act(self.ctx, self.slot_h, E, E, None, T, F, H, self.counts, self.offsets, self.xc, H, False,
                                      _DevPtr(self.slot_x.c.descale_snapshot), False, w_gateup8, w_gateup_descale, self.h8, F)
        else:
            gemm_fp8_nt_grouped(self.ctx, E, T, 2 * F, H, self.counts, self.offsets, self.xc, H, False,
                                _DevPtr(self.slot_x.c.descale_snapshot), False, w_gateup8, w_gateup_descale, self.gu, 2 * F)
            fp8_swiglu_quant_act(self.ctx, self.slot_h, self.gu, self.gu.view(-1)[F:], 2 * F, T, F, self.h8)
        gemm_fp8_nt_grouped(self.ctx, E, T, H, F, self.counts, self.offsets, self.h8, F, False,
                            _DevPtr(self.slot_h.c.descale_snapshot), False, w_down8, w_down_descale, self.yc, H)
        moe_combine_sorted_bf16(mixed, self.yc, route_weights, self.idx, self.counts, self.offsets, rows, E, H, accumulate)


class _DevPtr:
    """Wraps a raw device address so that it can be passed where a tensor is expected."""

    is_cuda = True

    def __init__(self, addr):
        self._addr = addr

    def data_ptr(self):
        return self._addr


class FfnSwigluFp8:
    """The reference's dense FP8 FFN (src/trainer.cu:6296-6322 and :7138-7146) with per-tensor delayed scaling:
    fp8_quant_act(x) -> gate and up GEMMs -> swiglu_forward -> fp8_quant_act -> down GEMM, here as three launches
    after the activation quantise: the gate/up GEMM carries SwiGLU and the re-quantise in its epilogue
    (cf_gemm_fp8_swiglu_quant_act), so the [M, 2F] bf16 intermediate is never written. `w_gateup8_interleaved` is the
    [2F, H] E4M3 tensor in the 32-row interleaved layout (fp8_interleave_gate_up), w_down8 is [H, F]."""

    def __init__(self, ctx, M, H, F, device="cuda"):
        self.ctx, self.M, self.H, self.F = ctx, M, H, F
        self.x8 = torch.empty((M, H), dtype=torch.uint8, device=device)
        self.h8 = torch.empty((M, F), dtype=torch.uint8, device=device)
        self.slot_x = ActSlot(ctx, E4M3_MAX)
        self.slot_h = ActSlot(ctx, E4M3_MAX)

    def forward(self, x, w_gateup8_interleaved, w_gateup_descale, w_down8, w_down_descale, y, bias=None, bias_mode=2):
        M, H, F = self.M, self.H, self.F
        fp8_quant_act(self.ctx, self.slot_x, x, self.x8)
        gemm_fp8_swiglu_quant_act(self.ctx, self.slot_h, 1, 1, None, M, F, H, None, None, self.x8, H, False,
                                  _DevPtr(self.slot_x.c.descale_snapshot), False, w_gateup8_interleaved, w_gateup_descale,
                                  self.h8, F)
        lt_gemm_fp8_nt(self.ctx, M, y.shape[1], F, self.h8, F, False, _DevPtr(self.slot_h.c.descale_snapshot), w_down8,
                       w_down_descale, y, y.stride(0), bias=bias, bias_mode=bias_mode)


class Fp8Block128Weight:
    """Weight [out, in] with its block-scaled cache: E4M3 codes and one scale per 128x128 block. The one cache serves the forward
    product (gemm_fp8_block128_nt) and the data gradient (gemm_fp8_block128_nn)."""

    def __init__(self, w):
        self.w = w                                       # bf16 master
        out_dim, in_dim = w.shape
        self.w8 = torch.empty((out_dim, (in_dim + 15) & ~15), dtype=torch.uint8, device=w.device)[:, :in_dim]
        self.descale = torch.empty((_blocks(out_dim), _blocks(in_dim)), dtype=torch.float32, device=w.device)
        self.refresh()

    def refresh(self):
        """Codes of the current master (after an optimiser step)."""
        fp8_quantize_block128x128(self.w, self.w8, self.descale)


class FfnSwigluFp8Block128:
    """Pre-norm SwiGLU feed-forward block on a residual stream with block-scaled FP8 products:
        h = x + residual;  n = rmsnorm(h) * gain;  g, u = n . w_gateup^T;  y = (silu(g) * u) . w_down^T
    `h` (the stream behind the addition) stays in self.h for the next layer. Up to max_rows rows a call: one token of a serving
    step as well as a training batch. train=True keeps what backward() needs; F must then be a multiple of 128. The column codes of n
    for the weight gradient are then taken from n's bf16 copy (one rounding more than the row codes have, and 2 + 2 bytes per element).
    Gradients are coded as E5M2 (grad_e5m2) or E4M3. The buffers belong to the object: one call at a time."""

    def __init__(self, ctx, max_rows, H, F, train=False, grad_e5m2=True, eps=1e-6, device="cuda"):
        if train and F % BLOCK:
            _refuse("FfnSwigluFp8Block128: training needs F to be a multiple of 128")
        self.ctx, self.H, self.F, self.train, self.e5m2, self.eps, self.max_rows = ctx, H, F, train, grad_e5m2, eps, max_rows
        R = max_rows

        def bf16(c):
            return torch.empty((R, c), dtype=torch.bfloat16, device=device)

        def codes(c):
            return torch.empty((R, (c + 15) & ~15), dtype=torch.uint8, device=device)[:, :c], block128_row_descale(R, c, device)

        def col_codes(c):
            return (torch.empty((R, (c + 15) & ~15), dtype=torch.uint8, device=device)[:, :c],
                    torch.empty((_blocks(R), c), dtype=torch.float32, device=device))

        self.h, self.gu, self.rms = bf16(H), bf16(2 * F), torch.empty(R, dtype=torch.float32, device=device)
        self.n8, self.a8 = codes(H), codes(F)
        if train:
            self.n, self.da, self.dn = bf16(H), bf16(F), bf16(H)
            self.n8c, self.a8c = col_codes(H), col_codes(F)
            self.dy8, self.dy8c, self.dgu8, self.dgu8c = codes(H), col_codes(H), codes(2 * F), col_codes(2 * F)
            self.scratch = torch.empty(add_rmsnorm_backward_scratch_floats(R, H), dtype=torch.float32, device=device)
        self.rows = None                                 # of the last forward() call that came through

    def _rows(self, pair):
        return pair[0][:self.rows], pair[1][:self.rows]

    def _cols(self, pair):
        return pair[0][:self.rows], pair[1][:_blocks(self.rows)]

    def forward(self, x, residual, gain, w_gateup, w_down, y):
        """x, y: bf16 [rows, H]; residual: bf16 [rows, H] or None; w_gateup: Fp8Block128Weight [2F, H] (gate rows first), w_down:
        [H, F]."""
        rows = x.shape[0]
        if rows > self.max_rows:
            _refuse(f"FfnSwigluFp8Block128: {rows} rows, made for {self.max_rows}")
        self.rows = rows
        try:
            self._forward(x, residual, gain, w_gateup, w_down, y)
        except BaseException:                            # what the call before it kept has been overwritten in part
            self.rows = None
            raise

    def _forward(self, x, residual, gain, w_gateup, w_down, y):
        rows = self.rows
        n8, dn8 = self._rows(self.n8)
        a8, da8 = self._rows(self.a8)
        gu = self.gu[:rows]
        add_rmsnorm_quantize_block128(x, residual, gain, self.h[:rows], self.rms[:rows], self.n[:rows] if self.train else None, n8, dn8,
                                      self.eps)
        gemm_fp8_block128_nt(self.ctx, n8, dn8, w_gateup.w8, w_gateup.descale, gu)
        gate, up = gu[:, :self.F], gu[:, self.F:]
        if self.train:
            n8c, dn8c = self._cols(self.n8c)
            fp8_quantize_block128(self.n[:rows], col8=n8c, col_descale=dn8c)
            a8c, da8c = self._cols(self.a8c)
            swiglu_quantize_block128(gate, up, a8, da8, a8c, da8c)
        else:
            swiglu_quantize_block128(gate, up, a8, da8)
        gemm_fp8_block128_nt(self.ctx, a8, da8, w_down.w8, w_down.descale, y)

    def backward(self, dy, dh, gain, w_gateup, w_down, dx, dw_gateup, dw_down, dgain, accumulate=False):
        """Gradients of the last forward() call for dy (of y) and dh (of the stream h, or None): dx (of x and residual alike),
        dw_gateup [2F, H], dw_down [H, F] (float32 or bf16), dgain (float32 [H]); the last three added to when accumulate."""
        if not self.train:
            _refuse("FfnSwigluFp8Block128: backward() needs train=True")
        if self.rows is None:
            _refuse("FfnSwigluFp8Block128: backward() needs a forward() call that came through")
        rows, F, e = self.rows, self.F, self.e5m2
        dy8, ddy8 = self._rows(self.dy8)
        dy8c, ddy8c = self._cols(self.dy8c)
        dgu8, ddgu8 = self._rows(self.dgu8)
        dgu8c, ddgu8c = self._cols(self.dgu8c)
        da, dn, gu = self.da[:rows], self.dn[:rows], self.gu[:rows]
        fp8_quantize_block128(dy, dy8, ddy8, dy8c, ddy8c, is_e5m2=e)
        gemm_fp8_block128_nn(self.ctx, dy8, ddy8, w_down.w8, w_down.descale, da, a_is_e5m2=e)
        gemm_fp8_block128_dw(self.ctx, dy8c, ddy8c, *self._cols(self.a8c), dw_down, x_is_e5m2=e, accumulate=accumulate)
        swiglu_backward_quantize_block128(gu[:, :F], gu[:, F:], da, dgu8, ddgu8, dgu8c, ddgu8c, is_e5m2=e)
        gemm_fp8_block128_nn(self.ctx, dgu8, ddgu8, w_gateup.w8, w_gateup.descale, dn, a_is_e5m2=e)
        gemm_fp8_block128_dw(self.ctx, dgu8c, ddgu8c, *self._cols(self.n8c), dw_gateup, x_is_e5m2=e, accumulate=accumulate)
        add_rmsnorm_backward(dn, self.h[:rows], gain, self.rms[:rows], dh, dx, dgain, self.scratch, accumulate)
