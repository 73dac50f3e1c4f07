"""ctypes bindings of libmllm_gpu.so.

``load_kernels()`` binds the drop-in symbols with exactly the ``argtypes``
the reference's Python engine uses for its C library
(src/mojollama/kernels/turbo_engine_v7_moe.py:_load_kernels, TE:240-392), so
engine code written against that library runs unchanged on this one.

``DeviceOps`` wraps the mllm_* device-pointer entry points for torch tensors
already on the GPU (the benchmark and batched paths).

There is no CPU fallback: if the library is missing or cannot be loaded,
``load_kernels()`` raises.
"""
import ctypes
import math
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libmllm_gpu.so")

cf = ctypes.POINTER(ctypes.c_float)
cu = ctypes.POINTER(ctypes.c_uint8)
ci = ctypes.c_int
cvp = ctypes.c_void_p

# Semantic ids (mllm_sem, mojollama_amd/csrc/mllm_common.h).
F32, Q4_0, Q4_1, Q5_0_F32, Q5_0_Q8, Q8_0, Q4_K_GGML, Q4_K_Q8 = range(8)
Q5_K_GGML, Q5_K_CE, Q6_K_GGML, Q6_K_LOWNIB, Q6_K_SEQ, MXFP4, MXFP4_CLAMP, MXFP4_Q8 = range(8, 16)
SEM_NAMES = ["F32", "Q4_0", "Q4_1", "Q5_0_F32", "Q5_0_Q8", "Q8_0", "Q4_K_GGML", "Q4_K_Q8",
             "Q5_K_GGML", "Q5_K_CE", "Q6_K_GGML", "Q6_K_LOWNIB", "Q6_K_SEQ", "MXFP4",
             "MXFP4_CLAMP", "MXFP4_Q8"]
# Reference entry points, for mllm_sem_for().
ENT_QMM, ENT_BMM, ENT_ROWS, ENT_MOE_GU, ENT_MOE_DOWN = range(5)


def build(verbose=False):
    """Compile libmllm_gpu.so for gfx950 in-tree (hipcc)."""
    r = subprocess.run(["make", "-s", "-C", os.path.join(HERE, "csrc")], capture_output=not verbose, text=True)
    if r.returncode != 0:
        raise RuntimeError("libmllm_gpu build failed:\n" + (r.stdout or "") + (r.stderr or ""))


class GemvFusion(ctypes.Structure):
    """mllm_gemv_fusion (include/mllm.h): the prologue/epilogue fused into a decode GEMV."""
    _fields_ = [("x_up", cvp), ("silu_clamp", ci), ("x_res", cvp), ("res_out", cvp), ("rms_w", cvp),
                ("rms_eps", ctypes.c_float), ("rms_div", ci), ("out_add", cvp), ("x_ld", ci), ("silu_pair", ci)]


class KVView(ctypes.Structure):
    """mllm_kv_view (include/mllm.h): a contiguous or paged KV cache on the device."""
    _fields_ = [("k", cvp), ("v", cvp), ("seq_stride", ctypes.c_long), ("block_tables", cvp), ("max_blocks", ci),
                ("page_size", ci), ("n_pages", ci)]


ATTN_CE, ATTN_GQA_C = 0, 1   # CE:141-158 gqa / gqa_attention.c:93 softmax

# Element types, and the layouts and scalings of rotary positions (include/mllm.h).
T_F32, T_F16, T_BF16, T_E4M3, T_I8 = range(5)
ROPE_HALF, ROPE_PAIRS = 0, 1
ROPE_NONE, ROPE_LINEAR, ROPE_NTK, ROPE_YARN, ROPE_BANDS = range(5)
_cl = ctypes.c_long


class PagedKV(ctypes.Structure):
    """mllm_paged_kv (include/mllm.h): a paged 16- or 8-bit KV cache."""
    _fields_ = [("type", ci), ("n_kv_head", ci), ("head_dim", ci), ("n_pages", ci), ("page_size", ci), ("k", cvp),
                ("v", cvp), ("k_exp", cvp), ("v_exp", cvp), ("page_stride", _cl), ("row_stride", _cl),
                ("head_stride", _cl), ("tables", cvp), ("n_seqs", ci), ("max_blocks", ci), ("table_ld", _cl)]


class Rotary(ctypes.Structure):
    """mllm_rotary (include/mllm.h): layout, width and frequencies of rotary positions."""
    _fields_ = [("layout", ci), ("rope_dim", ci), ("freqs", cvp), ("mscale", ctypes.c_float)]


class PageMap(ctypes.Structure):
    """mllm_page_map (include/mllm.h): which sequence holds which page."""
    _fields_ = [("tables", cvp), ("n_seqs", ci), ("max_blocks", ci), ("table_ld", _cl), ("refs", cvp), ("n_pages", ci),
                ("page_size", ci)]


class PagePlane(ctypes.Structure):
    """mllm_page_plane (include/mllm.h): memory that holds a slice of every page."""
    _fields_ = [("base", cvp), ("page_bytes", _cl), ("layer_bytes", _cl), ("n_layers", ci)]


class GptOssDesc(ctypes.Structure):
    """mllm_gptoss_desc (include/mllm.h): host pointers to gptoss_forward's weights."""
    _fields_ = [(n, ci) for n in ("L", "N", "NH", "NKH", "HD", "E", "K", "M", "max_ctx", "rope_dim", "outNR")] + [
        ("eps", ctypes.c_float), ("wQ", ctypes.POINTER(cu)), ("wK", ctypes.POINTER(cu)), ("wV", ctypes.POINTER(cu)),
        ("wO", ctypes.POINTER(cu)), ("wAN", ctypes.POINTER(cf)), ("wFN", ctypes.POINTER(cf)), ("wOut", cu),
        ("w_gate_inp", ctypes.POINTER(cf)), ("w_gate_exps", ctypes.POINTER(cu)), ("w_up_exps", ctypes.POINTER(cu)),
        ("w_down_exps", ctypes.POINTER(cu)), ("qt_gate", ci), ("qt_up", ci), ("qt_down", ci), ("cos_t", cf),
        ("sin_t", cf)]


# The reference caller's bindings of its whole-layer entry points, kept here
# so the drop-in and the reference's own C are called identically:
# ssm_layer_fused (TE:263-271, CE:803-849), qwen36_batch_forward (TE:273-310,
# CE:859-1231) and ssm_decode_step (TE:401-405, CE:736-802).
_pf, _pu, _pi = ctypes.POINTER(cf), ctypes.POINTER(cu), ctypes.POINTER(ci)
SSM_LAYER_FUSED_ARGTYPES = [cf, cf, cf, cf, cf, cf, cf, cf, cf, cf, cu, ci, ci, ci, cu, ci, ci, ci] + [ci] * 7
SSM_DECODE_STEP_ARGTYPES = [cf] * 9 + [ci] * 7
QWEN36_ARGTYPES = (
    [ci] * 7 + [ci, ci, ci, ctypes.c_float] + [ci] * 7        # B, L, N, NH, n_kv_h, HD, FF; E, K, M, eps; rope..dt_rank
    + [cf, ci]                                                # emb, emb_quant
    + [_pi, _pi, cf]                                          # layer_types, tokens, logits
    + [_pf, _pf]                                              # attn_norm_w, ffn_norm_w
    + [_pu, _pi, _pi, _pi] * 4                                # qkv, attn gate, ssm out, attn out: raw, nr, nc, qt
    + [_pu, _pi] * 3                                          # gate/up/down experts, quant types
    + [_pf, _pf, _pf, _pf, _pi]                               # shared expert gate/up/down, router, intermediate
    + [_pu, _pi, _pi, _pi, _pi]                               # moe router + qt, shared expert quant types
    + [cf, cu, ci, ci, ci]                                    # out_norm_w, out_w, nr, nc, qt
    + [_pf] * 6 + [cf]                                        # ssm conv1d, a, dt_bias, alpha, beta, norm; state
    + [cf, cf, _pi, cf, cf]                                   # kv_k, kv_v, kv_lens, cos_table, sin_table
    + [cf, cu])                                               # ws, q8_ws


def bind_model_entry_points(so):
    """Bind ssm_layer_fused / qwen36_batch_forward / ssm_decode_step as TE does."""
    so.ssm_layer_fused.argtypes = SSM_LAYER_FUSED_ARGTYPES
    so.ssm_layer_fused.restype = None
    so.qwen36_batch_forward.argtypes = QWEN36_ARGTYPES
    so.qwen36_batch_forward.restype = None
    so.ssm_decode_step.argtypes = SSM_DECODE_STEP_ARGTYPES
    so.ssm_decode_step.restype = None


_LIB = None


def load_kernels(path=LIB_PATH):
    """Load the library and bind the reference engine's symbols (TE:251-392) plus mllm_*."""
    global _LIB
    if _LIB is not None and path == LIB_PATH:
        return _LIB
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} is not built: run mojollama_amd.kernels.build() (needs hipcc)")
    # PyTorch-ROCm ships its own libamdhip64.so.7 and links it by another name.
    # Loading torch first makes this library bind to that same runtime, so one
    # HIP runtime serves both (and torch streams are valid handles here).
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    so = ctypes.CDLL(path)
    # --- as bound by TE:251-261, 363-377, 389-392
    so.quant_matmul_omp.argtypes = [cu, cf, cf, ci, ci, ci]
    so.quant_matmul_omp.restype = None
    so.f32_matmul_omp.argtypes = [cf, cf, cf, ci, ci]
    so.f32_matmul_omp.restype = None
    # QK:1139-1145 takes three quant types (TE:255 lists only two: its third is dropped there)
    so.batch_qkv_omp.argtypes = [cu, cu, cu, cf, cf, cf, cf, ci, ci, ci, ci, ci, ci, ci]
    so.batch_qkv_omp.restype = None
    so.batch_gate_up_omp.argtypes = [cu, cu, cf, cf, cf, ci, ci, ci, ci, ci]
    so.batch_gate_up_omp.restype = None
    so.set_num_threads.argtypes = [ci]
    so.set_num_threads.restype = None
    so.moe_forward_omp.argtypes = [ctypes.POINTER(cu), ctypes.POINTER(cu), ctypes.POINTER(cu), cf, ci, ci,
                                   ci, ci, ci, ctypes.POINTER(ctypes.c_int), cf, ci, cf, cf, cu]
    so.moe_forward_omp.restype = None
    for name in ("q6_k_dequantize_row", "q4_k_dequantize_row", "q5_k_dequantize_row", "q8_0_dequantize_row"):
        getattr(so, name).argtypes = [cu, cf, ci]
        getattr(so, name).restype = None
    # --- the engine's other kernel entry points (CE:68-534, 591; QK:1406, 1029)
    for name in ("q4_0_batch_matmul", "q8_0_batch_matmul", "q4_k_batch_matmul", "q6_k_batch_matmul",
                 "q5_k_batch_matmul", "mxfp4_batch_matmul"):
        getattr(so, name).argtypes = [cu, cf, cf, ci, ci, ci]
        getattr(so, name).restype = None
    bind_model_entry_points(so)
    so.moe_ffn.argtypes = [cvp, ci, cf, cf, cf, cf, ci]
    so.moe_ffn.restype = None
    so.moe_ffn_batched.argtypes = [cvp, ci, cf, cf, ci]
    so.moe_ffn_batched.restype = None
    so.quantize_row_q8_0.argtypes = [cf, cu, ci]
    so.quantize_row_q8_0.restype = ci
    so.get_max_threads.argtypes = []
    so.get_max_threads.restype = ci
    so.mllm_last_error.argtypes = []
    so.mllm_last_error.restype = ctypes.c_char_p
    so.mllm_cache_clear.argtypes = []
    so.mllm_cache_clear.restype = None
    # --- device-pointer API
    so.mllm_sem_for.argtypes = [ci, ci]
    so.mllm_sem_for.restype = ci
    so.mllm_raw_size.argtypes = [ci, ci, ci]
    so.mllm_raw_size.restype = ctypes.c_long
    so.mllm_packed_size.argtypes = [ci, ci, ci]
    so.mllm_packed_size.restype = ctypes.c_long
    so.mllm_pack.argtypes = [ci, cvp, cvp, ci, ci, cvp]
    so.mllm_pack.restype = ci
    so.mllm_gemv_workspace_size.argtypes = [ci, ci, ci, ci]
    so.mllm_gemv_workspace_size.restype = ctypes.c_long
    so.mllm_gemv.argtypes = [ci, cvp, cvp, cvp, ci, ci, ci, cvp, cvp]
    so.mllm_gemv.restype = ci
    so.mllm_gemv_fused_workspace_size.argtypes = [ci, ci, ci, ci, ctypes.POINTER(GemvFusion)]
    so.mllm_gemv_fused_workspace_size.restype = ctypes.c_long
    so.mllm_gemv_fused.argtypes = [ci, cvp, cvp, cvp, ci, ci, ci, ctypes.POINTER(GemvFusion), cvp, cvp]
    so.mllm_gemv_fused.restype = ci
    so.requantize_output_q8_0.argtypes = [cu, ci, ci, ci, cu]
    so.requantize_output_q8_0.restype = ci
    so.mllm_requantize_workspace_size.argtypes = [ci, ci, ci]
    so.mllm_requantize_workspace_size.restype = ctypes.c_long
    so.mllm_requantize_q8_0.argtypes = [ci, cvp, ci, ci, cvp, cvp, cvp]
    so.mllm_requantize_q8_0.restype = ci
    so.mllm_read_probe.argtypes = [cvp, ctypes.c_long, cvp, cvp]
    so.mllm_read_probe.restype = ci
    so.mllm_quantize_q8_0.argtypes = [cvp, ci, ci, cvp, cvp]
    so.mllm_quantize_q8_0.restype = ci
    so.mllm_router_packed_size.argtypes = [ci, ci]
    so.mllm_router_packed_size.restype = ctypes.c_long
    so.mllm_router_pack.argtypes = [cvp, ci, ci, cvp, cvp]
    so.mllm_router_pack.restype = ci
    so.mllm_route_workspace_size.argtypes = [ci, ci]
    so.mllm_route_workspace_size.restype = ctypes.c_long
    so.mllm_route.argtypes = [cvp, cvp, ci, ci, ci, ci, ci, cvp, cvp, cvp, cvp]
    so.mllm_route.restype = ci
    so.mllm_dequant.argtypes = [ci, cvp, ci, ci, cvp, cvp]
    so.mllm_dequant.restype = ci
    so.mllm_moe_dense_experts.argtypes = [cvp, cvp]
    so.mllm_moe_dense_experts.restype = ctypes.c_long
    so.mllm_moe_prepare.argtypes = [ci, ci, ci, ci, ci, ci, ci, ctypes.POINTER(cvp), ctypes.POINTER(cvp),
                                    ctypes.POINTER(cvp), cvp, ci]
    so.mllm_moe_prepare.restype = cvp
    so.mllm_moe_release.argtypes = [cvp]
    so.mllm_moe_release.restype = None
    so.mllm_moe_workspace_size.argtypes = [cvp, ci]
    so.mllm_moe_workspace_size.restype = ctypes.c_long
    so.mllm_moe_layer_info.argtypes = [cvp]
    so.mllm_moe_layer_info.restype = ci
    so.mllm_moe_forward.argtypes = [cvp, cvp, ci, cvp, cvp, ctypes.c_long, cvp, cvp, cvp]
    so.mllm_moe_forward.restype = ci
    so.mllm_moe_forward_noalloc.argtypes = [cvp, cvp, ci, cvp, cvp, cvp, cvp]
    so.mllm_moe_forward_noalloc.restype = ci
    so.mllm_moe_bucket.argtypes = [cvp, ci, ci, cvp, cvp, cvp, cvp, cvp]
    so.mllm_moe_bucket.restype = ci
    # --- decode attention and the KV cache (TE:383-385 binds gqa_attention_decode so)
    so.gqa_attention_decode.argtypes = [cf, cf, cf, cf, ci, ci, ci, ci, cf]
    so.gqa_attention_decode.restype = None
    so.mllm_gqa_workspace_size.argtypes = [ci, ci, ci, ci]
    so.mllm_gqa_workspace_size.restype = ctypes.c_long
    so.mllm_gqa_decode.argtypes = [ci, cvp, ctypes.POINTER(KVView), cvp, ci, ci, ci, ci, ci, cvp, cvp, ctypes.c_long,
                                   cvp]
    so.mllm_gqa_decode.restype = ci
    so.mllm_kv_append.argtypes = [ctypes.POINTER(KVView), cvp, cvp, cvp, ci, ci, ci, cvp]
    so.mllm_kv_append.restype = ci
    so.mllm_rope.argtypes = [cvp, ci, ci, ci, cvp, cvp, cvp, ci, cvp]
    so.mllm_rope.restype = ci
    # --- paged 16- or 8-bit KV cache: rotary positions, attention, pages
    pkv, pmap, pplane = ctypes.POINTER(PagedKV), ctypes.POINTER(PageMap), ctypes.POINTER(PagePlane)
    so.mllm_rotary_freqs.argtypes = [ci, ci] + [ctypes.c_double] * 5 + [ctypes.POINTER(ctypes.c_double), cf]
    so.mllm_rotary_freqs.restype = ci
    so.mllm_rotary_append.argtypes = ([ctypes.POINTER(Rotary), ci, cvp, _cl, cvp, _cl, cvp, _cl, cvp, ci, ci, ci, ci, ci,
                                       cvp, _cl, cvp, _cl, pkv, cvp, cvp, cvp])
    so.mllm_rotary_append.restype = ci
    so.mllm_paged_attn_workspace_size.argtypes = [pkv, ci, ci, ci, ci, ci]
    so.mllm_paged_attn_workspace_size.restype = _cl
    so.mllm_paged_attn_decode.argtypes = [pkv, ci, cvp, _cl, cvp, cvp, ci, ci, ci, ctypes.c_float, ci, cvp, ci, cvp,
                                          _cl, cvp, _cl, cvp]
    so.mllm_paged_attn_decode.restype = ci
    so.mllm_paged_attn_prompt.argtypes = [pkv, ci, cvp, _cl, cvp, cvp, cvp, ci, ci, ci, ci, ctypes.c_float, ci, cvp, ci,
                                          cvp, _cl, cvp, _cl, cvp]
    so.mllm_paged_attn_prompt.restype = ci
    so.mllm_pages_workspace_size.argtypes = [pmap, ci]
    so.mllm_pages_workspace_size.restype = _cl
    so.mllm_pages_reserve.argtypes = [pmap, ci, cvp, cvp, cvp, cvp, _cl, cvp]
    so.mllm_pages_reserve.restype = ci
    so.mllm_pages_free.argtypes = [pmap, ci, cvp, cvp, cvp]
    so.mllm_pages_free.restype = ci
    so.mllm_pages_fork.argtypes = [pmap, pplane, ci, ci, cvp, cvp, cvp, cvp, cvp, _cl, cvp]
    so.mllm_pages_fork.restype = ci
    so.mllm_pages_compact.argtypes = [pmap, pplane, ci, cvp, cvp, _cl, cvp]
    so.mllm_pages_compact.restype = ci
    so.mllm_pages_copy.argtypes = [pplane, ci, ci, ci, cvp, cvp, cvp]
    so.mllm_pages_copy.restype = ci
    # --- layers in 8-bit integers
    so.mllm_i8_quantize.argtypes = [ci, cvp, _cl, ci, ci, cvp, _cl, cvp, cvp]
    so.mllm_i8_quantize.restype = ci
    so.mllm_i8_dequant.argtypes = [cvp, _cl, cvp, ci, ci, ci, cvp, _cl, cvp]
    so.mllm_i8_dequant.restype = ci
    so.mllm_i8_rms_norm.argtypes = [ci, cvp, _cl, ci, cvp, _cl, cvp, _cl, ci, cvp, ctypes.c_float, ci, ci, cvp, _cl, cvp,
                                    cvp]
    so.mllm_i8_rms_norm.restype = ci
    so.mllm_i8_silu_mul.argtypes = [ci, cvp, _cl, cvp, _cl, ci, ci, cvp, _cl, cvp, cvp]
    so.mllm_i8_silu_mul.restype = ci
    so.mllm_i8_packed_size.argtypes = [ci, ci]
    so.mllm_i8_packed_size.restype = _cl
    so.mllm_i8_pack.argtypes = [ci, cvp, _cl, ci, ci, cvp, cvp, cvp]
    so.mllm_i8_pack.restype = ci
    so.mllm_i8_gemm_workspace_size.argtypes = [ci, ci, ci]
    so.mllm_i8_gemm_workspace_size.restype = _cl
    so.mllm_i8_gemm.argtypes = [cvp, cvp, cvp, _cl, cvp, ci, ci, ci, cvp, ci, cvp, _cl, cvp, _cl, cvp]
    so.mllm_i8_gemm.restype = ci
    # gptoss_forward (GO:96-130 argument list)
    pcu, pcf, pci = ctypes.POINTER(cu), ctypes.POINTER(cf), ctypes.POINTER(ci)
    so.gptoss_forward.argtypes = ([pci, ci, cf, ci] + [pcu] * 4 + [pcf] * 2 + [pci] * 8 + [cu, ci, ci, ci, cf, cf, pci,
                                  cf, cf, ci, ci, cf, ci] + [ci] * 6 + [ctypes.c_float] + [ci] * 3 + [pcf] +
                                  [pcu] * 3 + [ci] * 3 + [cf, cf, cu, cf])
    so.gptoss_forward.restype = None
    so.mllm_gptoss_create.argtypes = [cvp]
    so.mllm_gptoss_create.restype = cvp
    so.mllm_gptoss_release.argtypes = [cvp]
    so.mllm_gptoss_release.restype = None
    so.mllm_gptoss_kv_floats.argtypes = [cvp]
    so.mllm_gptoss_kv_floats.restype = ctypes.c_long
    so.mllm_gptoss_step.argtypes = [cvp, cvp, cvp, cvp, cvp, cvp, cvp, cvp]
    so.mllm_gptoss_step.restype = ci
    so.mllm_page_table_create.argtypes = [ci, ci]
    so.mllm_page_table_create.restype = cvp
    so.mllm_page_table_destroy.argtypes = [cvp]
    so.mllm_page_table_destroy.restype = None
    so.mllm_page_table_alloc.argtypes = [cvp]
    so.mllm_page_table_alloc.restype = ci
    so.mllm_page_table_free.argtypes = [cvp, ci]
    so.mllm_page_table_free.restype = None
    so.mllm_page_table_map.argtypes = [cvp, ci, ci]
    so.mllm_page_table_map.restype = None
    so.mllm_page_table_lookup.argtypes = [cvp, ci]
    so.mllm_page_table_lookup.restype = ci
    so.mllm_page_table_entries.argtypes = [cvp]
    so.mllm_page_table_entries.restype = ctypes.POINTER(ci)
    if path == LIB_PATH:
        _LIB = so
    return so


def last_error(so=None):
    so = so or load_kernels()
    return so.mllm_last_error().decode()


class DeviceOps:
    """mllm_* calls on torch tensors that live on the current GPU."""

    def __init__(self, so=None):
        import torch
        self.torch = torch
        self.so = so or load_kernels()
        # the current device as the runtime has it (no call here makes it the first to ask: tensors are there by then)
        self._cur_raw = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        self._stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", lambda cur: torch.cuda.current_stream(cur).cuda_stream)
        self._int8, self._f32 = torch.int8, torch.float32
        self._reals = {torch.float32: T_F32, torch.float16: T_F16, torch.bfloat16: T_BF16}
        self._types = {torch.float32: T_F32, torch.float16: T_F16, torch.bfloat16: T_BF16, torch.float8_e4m3fn: T_E4M3}

    def _stream(self):
        return ctypes.c_void_p(self.torch.cuda.current_stream().cuda_stream)

    def _check(self, rc, what):
        if rc != 0:
            raise RuntimeError(f"{what} failed: {last_error(self.so)}")

    def pack(self, sem, raw_dev, n_rows, n_cols):
        """raw GGUF bytes (uint8 tensor on GPU) -> packed uint8 tensor."""
        torch = self.torch
        n = self.so.mllm_packed_size(sem, n_rows, n_cols)
        packed = torch.empty(n, dtype=torch.uint8, device=raw_dev.device)
        self._check(self.so.mllm_pack(sem, raw_dev.data_ptr(), packed.data_ptr(), n_rows, n_cols, self._stream()),
                    "mllm_pack")
        return packed

    def workspace(self, sem, n_cols, B, device, n_rows=0):
        n = self.so.mllm_gemv_workspace_size(sem, n_rows, n_cols, B)
        return self.torch.empty(max(n, 256), dtype=self.torch.uint8, device=device) if n > 0 else None

    def gemv(self, sem, packed, x, n_rows, n_cols, out=None, ws=None):
        torch = self.torch
        B = x.numel() // n_cols
        if out is None:
            out = torch.empty((B, n_rows), dtype=torch.float32, device=x.device)
        if ws is None:
            ws = self.workspace(sem, n_cols, B, x.device, n_rows)
        self._check(self.so.mllm_gemv(sem, packed.data_ptr(), x.data_ptr(), out.data_ptr(), n_rows, n_cols, B,
                                      ws.data_ptr() if ws is not None else None, self._stream()), "mllm_gemv")
        return out

    def fusion(self, x_up=None, silu_clamp=True, x_res=None, res_out=None, rms_w=None, rms_eps=1e-6, rms_div=False,
               out_add=None, x_ld=0, silu_pair=False):
        """An mllm_gemv_fusion over torch tensors or device addresses (None = field unused)."""
        p = lambda t: (t if isinstance(t, int) else t.data_ptr()) if t is not None else None  # noqa: E731
        return GemvFusion(p(x_up), int(silu_clamp), p(x_res), p(res_out), p(rms_w), float(rms_eps), int(rms_div),
                          p(out_add), int(x_ld), int(silu_pair))

    def gemv_fused(self, sem, packed, x, n_rows, n_cols, fusion, out=None, ws=None, B=None):
        """mllm_gemv_fused: y = W * prologue(x) (+ out_add), one launch where it fits.
        x: a tensor, or a device address with B given (a strided view inside a wider row)."""
        torch = self.torch
        if B is None:
            B = x.numel() // n_cols
        xp = x if isinstance(x, int) else x.data_ptr()
        dev = torch.device("cuda")
        if out is None:
            out = torch.empty((B, n_rows), dtype=torch.float32, device=dev)
        if ws is None:
            n = self.so.mllm_gemv_fused_workspace_size(sem, n_rows, n_cols, B, ctypes.byref(fusion))
            ws = torch.empty(max(n, 256), dtype=torch.uint8, device=dev) if n > 0 else None
        self._check(self.so.mllm_gemv_fused(sem, packed.data_ptr(), xp, out.data_ptr(), n_rows, n_cols, B,
                                            ctypes.byref(fusion), ws.data_ptr() if ws is not None else None,
                                            self._stream()), "mllm_gemv_fused")
        return out

    def quantize_q8_0(self, x, n_cols):
        torch = self.torch
        T = x.numel() // n_cols
        q8 = torch.empty(T * (n_cols // 32) * 34, dtype=torch.uint8, device=x.device)
        self._check(self.so.mllm_quantize_q8_0(x.data_ptr(), T, n_cols, q8.data_ptr(), self._stream()),
                    "mllm_quantize_q8_0")
        return q8

    def router_pack(self, router):
        """fp32 router [E][N] (device) -> the routing layout (mllm_router_pack)."""
        torch = self.torch
        E, N = router.shape
        out = torch.empty(self.so.mllm_router_packed_size(N, E) // 4, dtype=torch.float32, device=router.device)
        self._check(self.so.mllm_router_pack(router.data_ptr(), N, E, out.data_ptr(), self._stream()),
                    "mllm_router_pack")
        return out

    def route(self, router, x, K, renorm, packed=None, slices=True):
        """Top-K routing of x [T][N] by the fp32 router [E][N] (device); slices=False
        keeps one workgroup per token at T <= 8 (no workspace)."""
        torch = self.torch
        E, N = router.shape
        rp = self.router_pack(router) if packed is None else packed
        T = x.numel() // N
        idx = torch.empty((T, K), dtype=torch.int32, device=x.device)
        w = torch.empty((T, K), dtype=torch.float32, device=x.device)
        ws = torch.empty(self.so.mllm_route_workspace_size(T, E) // 4, dtype=torch.float32, device=x.device) \
            if slices else None
        self._check(self.so.mllm_route(rp.data_ptr(), x.data_ptr(), T, N, E, K, int(renorm), idx.data_ptr(),
                                       w.data_ptr(), ws.data_ptr() if ws is not None else None, self._stream()),
                    "mllm_route")
        return idx, w

    def dequant(self, sem, packed, n_rows, n_cols):
        torch = self.torch
        out = torch.empty((n_rows, n_cols), dtype=torch.float32, device=packed.device)
        self._check(self.so.mllm_dequant(sem, packed.data_ptr(), n_rows, n_cols, out.data_ptr(), self._stream()),
                    "mllm_dequant")
        return out

    # ------------------------------------------------------------ MoE layer
    def kv_view(self, k, v, seq_stride=0, block_tables=None, page_size=0, n_pages=0):
        """An mllm_kv_view over fp32 GPU tensors k, v (block_tables: int32 [B][max_blocks] GPU).
        The view keeps the tensors alive."""
        view = KVView(k.data_ptr(), v.data_ptr(), int(seq_stride),
                      block_tables.data_ptr() if block_tables is not None else None,
                      int(block_tables.shape[-1]) if block_tables is not None else 0, int(page_size), int(n_pages))
        view._tensors = (k, v, block_tables)
        return view

    def gqa_decode(self, mode, q, kv, seq_lens, max_seq, NH, NKH, HD, out=None, ws=None):
        """mllm_gqa_decode: q [B][NH*HD] fp32, seq_lens int32 [B] (GPU)."""
        torch = self.torch
        B = q.numel() // (NH * HD)
        if out is None:
            out = torch.empty((B, NH * HD), dtype=torch.float32, device=q.device)
        n = self.so.mllm_gqa_workspace_size(B, NH, HD, max_seq)
        if ws is None:
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        self._check(self.so.mllm_gqa_decode(mode, q.data_ptr(), ctypes.byref(kv), seq_lens.data_ptr(), max_seq, B, NH,
                                            NKH, HD, out.data_ptr(), ws.data_ptr(), ws.numel(), self._stream()),
                    "mllm_gqa_decode")
        return out

    def kv_append(self, kv, pos, k_new, v_new, NKH, HD):
        B = pos.numel()
        self._check(self.so.mllm_kv_append(ctypes.byref(kv), pos.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), B,
                                           NKH, HD, self._stream()), "mllm_kv_append")

    def rope(self, buf, NH, HD, pos, cos_t, sin_t, rope_dim=0):
        T = pos.numel()
        self._check(self.so.mllm_rope(buf.data_ptr(), T, NH, HD, pos.data_ptr(), cos_t.data_ptr(), sin_t.data_ptr(),
                                      rope_dim, self._stream()), "mllm_rope")
        return buf

    # ------------------------------------------- paged 16- or 8-bit KV cache
    def _cur(self):
        return self.torch.cuda.current_device()

    def _raw_stream(self, cur):
        return self._stream_of(cur)

    def _type(self, t, what, cur):
        """mllm type of a tensor on the current GPU (cur) whose last dimension is dense."""
        code = self._types.get(t.dtype)
        if code is None:
            raise TypeError(f"{what}: {t.dtype} is not served")
        if t.get_device() != cur:
            self._elsewhere(t, what)
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise ValueError(f"{what}: the last dimension is not dense")
        return code

    def _elsewhere(self, t, what):
        raise ValueError(f"{what}: a tensor on {t.device}, not on the current GPU")

    def _room(self, ws, cur):
        """A workspace's address and bytes are what its entry writes to: on the current GPU (cur), with nothing between."""
        if ws.get_device() != cur:
            self._elsewhere(ws, "workspace")
        if not ws.is_contiguous():
            raise ValueError("workspace: a dense tensor is needed")

    @staticmethod
    def _made_here(cur, *handles):
        for h in handles:
            if h is not None and h._device != cur:
                raise ValueError(f"a {type(h).__name__} of GPU {h._device}, not of the current one")

    def _ints(self, t, what, cur, n=None):
        """Address of a dense int32 tensor on the current GPU (None: a null pointer)."""
        if t is None:
            return None
        if t.get_device() != cur:
            self._elsewhere(t, what)
        if t.dtype != self.torch.int32 or not t.is_contiguous() or (n is not None and t.numel() != n):
            raise ValueError(f"{what}: a dense int32 tensor{'' if n is None else ' of %d' % n} is needed")
        return t.data_ptr()

    def paged_kv(self, k, v, tables, k_exp=None, v_exp=None):
        """An mllm_paged_kv over pools k, v [n_pages, page_size, n_kv_head, head_dim] (float16, bfloat16 or
        float8_e4m3fn; any strides, the last dimension dense, so a [page][head][row] pool is passed permuted) and
        tables int32 [n_seqs, max_blocks]; float8 pools with their exponents uint8 [n_pages, n_kv_head, page_size].
        The view keeps the tensors alive."""
        torch, cur = self.torch, self._cur()
        code = self._type(k, "k", cur)
        if code != self._type(v, "v", cur) or k.shape != v.shape or k.stride() != v.stride() or k.dim() != 4:
            raise ValueError("k and v: two pools [page, row, head, element] of one type, shape and strides")
        if tables.get_device() != cur:
            self._elsewhere(tables, "tables")
        if tables.dtype != torch.int32 or tables.dim() != 2 or tables.stride(1) != 1:
            raise ValueError("tables: int32 [n_seqs, max_blocks], rows dense")
        n_pages, page, heads, hd = k.shape
        for e in (k_exp, v_exp):
            if (e is None) != (code != T_E4M3):
                raise ValueError("k_exp and v_exp belong to float8 pools")
            if e is not None:
                if e.get_device() != cur:
                    self._elsewhere(e, "exponents")
                if e.dtype != torch.uint8 or tuple(e.shape) != (n_pages, heads, page) or not e.is_contiguous():
                    raise ValueError("exponents: dense uint8 [n_pages, n_kv_head, page_size]")
        p = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        view = PagedKV(code, heads, hd, n_pages, page, p(k), p(v), p(k_exp), p(v_exp), k.stride(0), k.stride(1),
                       k.stride(2), p(tables), tables.shape[0], tables.shape[1], tables.stride(0))
        view._tensors, view._device = (k, v, tables, k_exp, v_exp), cur
        return view

    def rotary(self, rope_dim, layout=ROPE_HALF, base=10000.0, scaling=ROPE_NONE, factor=1.0, ctx=0.0, beta_fast=0.0,
               beta_slow=0.0, freqs=None, mscale=None):
        """An mllm_rotary with its frequencies on the current GPU: those of mllm_rotary_freqs, or the caller's own
        rope_dim / 2 (freqs, radians per position, in place of a scaling).  mscale None: the scaling's factor."""
        torch = self.torch
        if freqs is None:
            f, m = (ctypes.c_double * max(rope_dim // 2, 1))(), ctypes.c_float()
            self._check(self.so.mllm_rotary_freqs(scaling, rope_dim, base, factor, ctx, beta_fast, beta_slow, f,
                                                  ctypes.byref(m)), "mllm_rotary_freqs")
            freqs, scale = torch.tensor(list(f), dtype=torch.float64), m.value
        else:
            freqs, scale = torch.as_tensor(freqs, dtype=torch.float64, device="cpu"), 1.0
            if scaling != ROPE_NONE or rope_dim % 2 or tuple(freqs.shape) != (rope_dim // 2,) or not freqs.isfinite().all():
                raise ValueError("freqs: rope_dim / 2 finite frequencies, in place of a scaling")
        if mscale is not None:
            scale = float(mscale)
            if not math.isfinite(scale):
                raise ValueError("mscale is finite")
        freqs = freqs.cuda()
        rot = Rotary(layout, rope_dim, freqs.data_ptr(), scale)
        rot._tensors, rot._device = (freqs,), self._cur()
        return rot

    def rotary_append(self, rot, q, k, v, pos, NH=0, NKH=0, HD=0, kv=None, seqs=None, rows=None, q_out=None, k_out=None):
        """mllm_rotary_append: q [T, NH*HD], k, v [T, NKH*HD] (parts of a fused buffer may be passed as slices; q, or k
        and v, may be None), pos int32 [T]; k and v go to rows `rows` (None: pos) of sequences `seqs` (None: 0, 1, ...)
        of kv, the turned q to q_out and k to k_out.  Heads and head size come from kv where it is given."""
        cur = self._cur()
        self._made_here(cur, rot, kv)
        pp, T = self._ints(pos, "pos", cur), pos.numel()
        if kv is not None:
            NKH, HD = kv.n_kv_head, kv.head_dim
        it, qp, ql = self._rows(q, "q", T, NH * HD, cur, None)
        it, kp, kl = self._rows(k, "k", T, NKH * HD, cur, it)
        it, vp, vl = self._rows(v, "v", T, NKH * HD, cur, it)
        ot, qop, qol = self._rows(q_out, "q_out", T, NH * HD, cur, None)
        ot, kop, kol = self._rows(k_out, "k_out", T, NKH * HD, cur, ot)
        self._check(self.so.mllm_rotary_append(
            rot, it or T_F32, qp, ql, kp, kl, vp, vl, pp, T, NH, NKH, HD, ot or T_F32, qop, qol, kop, kol, kv,
            self._ints(seqs, "seqs", cur, T), self._ints(rows, "rows", cur, T), self._raw_stream(cur)),
            "mllm_rotary_append")

    def _rows(self, t, what, T, n, cur, code):
        """(type, address, row stride) of a [T, n] tensor of type `code` (None: any); nothing for None."""
        if t is None:
            return code, None, 0
        c = self._type(t, what, cur)
        if t.dim() != 2 or t.shape[0] != T or t.shape[1] != n:
            raise ValueError(f"{what}: [{T}, {n}] is needed, got {list(t.shape)}")
        if code is not None and c != code:
            raise TypeError("q, k and v have one type, and q_out and k_out")
        return c, t.data_ptr(), t.stride(0) if T > 1 else max(t.stride(0), n)

    def paged_attn_workspace(self, kv, T, B, NH, max_len, window=0):
        """A workspace for paged_attn_decode (T = B) and paged_attn_prompt calls up to these sizes."""
        n = self.so.mllm_paged_attn_workspace_size(kv, T, B, NH, max_len, window)
        if n < 0:
            raise ValueError("paged_attn_workspace: sizes that are not served")
        return self.torch.empty(n, dtype=self.torch.uint8, device="cuda")

    def _attn(self, kv, q, T, B, NH, max_len, window, sinks, out, out_dtype, ws, cur):
        self._made_here(cur, kv)
        n = NH * kv.head_dim
        qt, qp, ql = self._rows(q, "q", T, n, cur, None)
        if out is None:
            out = self.torch.empty((T, n), dtype=out_dtype or q.dtype, device=q.device)
        ot, op, ol = self._rows(out, "out", T, n, cur, None)
        sk = None
        if sinks is not None:
            if sinks.get_device() != cur:
                self._elsewhere(sinks, "sinks")
            if sinks.dtype != self.torch.float32 or sinks.numel() != NH or not sinks.is_contiguous():
                raise ValueError("sinks: dense float32 [NH]")
            sk = sinks.data_ptr()
        if ws is None:
            ws = self.paged_attn_workspace(kv, T, B, NH, max_len, window)
        else:
            self._room(ws, cur)
        return qt, qp, ql, out, ot, op, ol, ws, sk

    def paged_attn_decode(self, kv, q, lens, max_len, NH, scale=None, window=0, sinks=None, seqs=None, out=None,
                          out_dtype=None, ws=None):
        """mllm_paged_attn_decode: q [B, NH*HD], lens int32 [B] (cached rows, the new one among them, at most max_len);
        scale None: 1/sqrt(HD); out in out_dtype (None: q's)."""
        B, cur = q.shape[0], self._cur()
        qt, qp, ql, out, ot, op, ol, ws, sk = self._attn(kv, q, B, B, NH, max_len, window, sinks, out, out_dtype, ws, cur)
        self._check(self.so.mllm_paged_attn_decode(
            kv, qt, qp, ql, self._ints(seqs, "seqs", cur, B), self._ints(lens, "lens", cur, B), max_len, B, NH,
            kv.head_dim ** -0.5 if scale is None else scale, window, sk, ot, op, ol, ws.data_ptr(), ws.nbytes,
            self._raw_stream(cur)), "mllm_paged_attn_decode")
        return out

    def paged_attn_prompt(self, kv, q, starts, lens, max_len, NH, scale=None, window=0, sinks=None, seqs=None, out=None,
                          out_dtype=None, ws=None):
        """mllm_paged_attn_prompt: q [T, NH*HD] holds the new tokens of B sequences, starts int32 [B + 1], lens int32
        [B] (cached rows, the new ones among them, at most max_len)."""
        T, B, cur = q.shape[0], lens.numel(), self._cur()
        qt, qp, ql, out, ot, op, ol, ws, sk = self._attn(kv, q, T, B, NH, max_len, window, sinks, out, out_dtype, ws, cur)
        self._check(self.so.mllm_paged_attn_prompt(
            kv, qt, qp, ql, self._ints(seqs, "seqs", cur, B), self._ints(starts, "starts", cur, B + 1),
            self._ints(lens, "lens", cur, B), max_len, T, B, NH, kv.head_dim ** -0.5 if scale is None else scale, window,
            sk, ot, op, ol, ws.data_ptr(), ws.nbytes, self._raw_stream(cur)), "mllm_paged_attn_prompt")
        return out

    def page_map(self, tables, refs, page_size):
        """An mllm_page_map over tables int32 [n_seqs, max_blocks] (-1 unmapped) and refs int32 [n_pages]."""
        cur = self._cur()
        if tables.get_device() != cur:
            self._elsewhere(tables, "tables")
        if tables.dtype != self.torch.int32 or tables.dim() != 2 or tables.stride(1) != 1:
            raise ValueError("tables: int32 [n_seqs, max_blocks], rows dense")
        m = PageMap(tables.data_ptr(), tables.shape[0], tables.shape[1], tables.stride(0), self._ints(refs, "refs", cur),
                    refs.numel(), page_size)
        m._tensors, m._device = (tables, refs), cur
        return m

    def page_planes(self, pools):
        """mllm_page_plane entries of pools [n_layers, n_pages, ...], each layer's pages dense (K, V, and the exponents
        of float8 pools)."""
        planes = (PagePlane * len(pools))()
        for p, t in zip(planes, pools):
            if t.get_device() != self._cur():
                self._elsewhere(t, "pool")
            if t.dim() < 2 or not t[0].is_contiguous():
                raise ValueError("pools: [n_layers, n_pages, ...], each layer dense")
            p.base, p.n_layers = t.data_ptr(), t.shape[0]
            p.page_bytes, p.layer_bytes = t.stride(1) * t.element_size(), t.stride(0) * t.element_size()
        planes._tensors, planes._n_pages = tuple(pools), min((t.shape[1] for t in pools), default=None)
        planes._device = self._cur()
        return planes

    def pages_workspace(self, m, n):
        """A workspace for pages_reserve and pages_fork calls of up to n requests, and pages_compact."""
        return self.torch.empty(self.so.mllm_pages_workspace_size(m, n), dtype=self.torch.uint8, device="cuda")

    def _pages_args(self, m, n, status, ws, cur):
        torch = self.torch
        self._made_here(cur, m)
        if status is None:
            status = torch.empty(1, dtype=torch.int32, device="cuda")
        if ws is None:
            ws = self.pages_workspace(m, n)
        else:
            self._room(ws, cur)
        return status, self._ints(status, "status", cur, 1), ws

    def _pages_in(self, planes, n_pages, cur):
        self._made_here(cur, planes)
        if planes._n_pages is not None and planes._n_pages < n_pages:
            raise ValueError(f"a pool holds {planes._n_pages} pages, not {n_pages}")

    def pages_reserve(self, m, seqs, lens, status=None, ws=None):
        """mllm_pages_reserve: pages for rows below lens[i] of sequences seqs[i]; returns status (a device int32, 0 when
        every request was met)."""
        n, cur = seqs.numel(), self._cur()
        status, sp, ws = self._pages_args(m, n, status, ws, cur)
        self._check(self.so.mllm_pages_reserve(m, n, self._ints(seqs, "seqs", cur), self._ints(lens, "lens", cur, n), sp,
                                               ws.data_ptr(), ws.nbytes, self._raw_stream(cur)),
                    "mllm_pages_reserve")
        return status

    def pages_free(self, m, seqs, lens=None):
        """mllm_pages_free: sequences seqs[i] give back their pages past the first lens[i] rows (None: all)."""
        n, cur = seqs.numel(), self._cur()
        self._made_here(cur, m)
        self._check(self.so.mllm_pages_free(m, n, self._ints(seqs, "seqs", cur), self._ints(lens, "lens", cur, n),
                                            self._raw_stream(cur)), "mllm_pages_free")

    def pages_fork(self, m, planes, parents, children, lens, status=None, ws=None):
        """mllm_pages_fork: children[i] takes over the first lens[i] rows of parents[i], all at once; returns status."""
        n, cur = parents.numel(), self._cur()
        self._pages_in(planes, m.n_pages, cur)
        status, sp, ws = self._pages_args(m, n, status, ws, cur)
        self._check(self.so.mllm_pages_fork(m, planes, len(planes), n, self._ints(parents, "parents", cur),
                                            self._ints(children, "children", cur, n), self._ints(lens, "lens", cur, n), sp,
                                            ws.data_ptr(), ws.nbytes, self._raw_stream(cur)),
                    "mllm_pages_fork")
        return status

    def pages_compact(self, m, planes, status=None, ws=None):
        """mllm_pages_compact: the live pages move to the front; returns their number (a device int32)."""
        cur = self._cur()
        self._pages_in(planes, m.n_pages, cur)
        status, sp, ws = self._pages_args(m, 0, status, ws, cur)
        self._check(self.so.mllm_pages_compact(m, planes, len(planes), sp, ws.data_ptr(),
                                               ws.nbytes, self._raw_stream(cur)), "mllm_pages_compact")
        return status

    def pages_copy(self, planes, n_pages, src, dst):
        """mllm_pages_copy: page dst[i] := page src[i] in every plane."""
        n, cur = src.numel(), self._cur()
        self._pages_in(planes, n_pages, cur)
        self._check(self.so.mllm_pages_copy(planes, len(planes), n_pages, n, self._ints(src, "src", cur),
                                            self._ints(dst, "dst", cur, n), self._raw_stream(cur)), "mllm_pages_copy")

    # ------------------------------------------- layers in 8-bit integers
    # (a call's own time is that of a launch, so the checks of a tensor that is as it should be are few)
    def _real(self, t, what):
        """mllm type of a float32, float16 or bfloat16 tensor."""
        code = self._reals.get(t.dtype)
        if code is None:
            raise TypeError(f"{what}: {t.dtype} is not served")
        return code

    def _at(self, t, what, cur, T, n):
        """(address, row stride) of a [T, n] tensor on the current GPU (cur) whose last dimension is dense."""
        if t.shape != (T, n) or t.get_device() != cur:
            if t.get_device() != cur:
                self._elsewhere(t, what)
            raise ValueError(f"{what}: [{T}, {n}] is needed, got {list(t.shape)}")
        ld, dense = t.stride()
        if dense != 1 and n > 1:
            raise ValueError(f"{what}: the last dimension is not dense")
        return t.data_ptr(), ld if T > 1 else n

    def _codes(self, t, what, cur, T, n):
        """_at of int8."""
        if t.dtype != self._int8:
            raise TypeError(f"{what}: {t.dtype}, not int8")
        return self._at(t, what, cur, T, n)

    def _floats(self, t, what, cur, n):
        """Address of a dense float32 [n] tensor on the current GPU (None: a null pointer)."""
        if t is None:
            return None
        if t.dtype != self._f32 or t.numel() != n or not t.is_contiguous() or t.get_device() != cur:
            if t.get_device() != cur:
                self._elsewhere(t, what)
            raise ValueError(f"{what}: dense float32 [{n}]")
        return t.data_ptr()

    @staticmethod
    def _sizes(t, what):
        s = t.shape
        if len(s) != 2:
            raise ValueError(f"{what}: [tokens, elements], got {list(s)}")
        T, n = s
        if T > 1073741824 or n > 1073741824:     # the entries take 32-bit sizes
            raise ValueError(f"{what}: at most 2^30 in each dimension, got {list(s)}")
        return T, n

    def _i8_new(self, q, scale, T, n):
        """The outputs of the calls that quantise, where they are not given: rows of codes at multiples of 16 bytes, as
        i8_gemm takes them; long ones at whole lines (1000 tokens x 2048 x 2048: 9.5 us, 9.9 with rows 16 bytes off)."""
        if q is None:
            step = 128 if n >= 1024 else 16
            q = self.torch.empty((T, (n + step - 1) // step * step), dtype=self._int8, device="cuda")[:, :n]
        if scale is None:
            scale = self.torch.empty(T, dtype=self._f32, device="cuda")
        return q, scale

    def i8_quantize(self, x, q=None, scale=None):
        """mllm_i8_quantize: x [T, n] (float32, float16 or bfloat16) -> (q int8 [T, n], scale float32 [T])."""
        cur, xt = self._cur_raw(), self._real(x, "x")
        T, n = self._sizes(x, "x")
        xp, xl = self._at(x, "x", cur, T, n)
        if q is None or scale is None:
            q, scale = self._i8_new(q, scale, T, n)
        qp, ql = self._codes(q, "q", cur, T, n)
        sp = self._floats(scale, "scale", cur, T)
        rc = self.so.mllm_i8_quantize(xt, xp, xl, T, n, qp, ql, sp, self._stream_of(cur))
        if rc:
            self._check(rc, "mllm_i8_quantize")
        return q, scale

    def i8_dequant(self, q, scale, out=None, out_dtype=None):
        """mllm_i8_dequant: scale[t] * q[t] in out_dtype (None: bfloat16)."""
        cur = self._cur_raw()
        T, n = self._sizes(q, "q")
        qp, ql = self._codes(q, "q", cur, T, n)
        if out is None:
            out = self.torch.empty((T, n), dtype=out_dtype or self.torch.bfloat16, device="cuda")
        ot = self._real(out, "out")
        op, ol = self._at(out, "out", cur, T, n)
        rc = self.so.mllm_i8_dequant(qp, ql, self._floats(scale, "scale", cur, T), T, n, ot, op, ol, self._stream_of(cur))
        if rc:
            self._check(rc, "mllm_i8_dequant")
        return out

    def i8_rms_norm(self, x, w, eps, res=None, res_out=None, q=None, scale=None):
        """mllm_i8_rms_norm: x [T, n] plus the residual stream res (None: none), which goes on in res_out (None: res
        itself), normed with w [n] -> (q, scale)."""
        cur, xt, wt = self._cur_raw(), self._real(x, "x"), self._real(w, "w")
        T, n = self._sizes(x, "x")
        xp, xl = self._at(x, "x", cur, T, n)
        rt = rl = ol = 0
        rp = op = None
        if res is not None:
            rt = self._real(res, "res")
            rp, rl = self._at(res, "res", cur, T, n)
            if res_out is None:
                op, ol = rp, rl
            else:
                op, ol = self._at(res_out, "res_out", cur, T, n)
                if res_out.dtype != res.dtype:
                    raise TypeError("res and res_out have one type")
        elif res_out is not None:
            raise ValueError("res_out belongs to res")
        if w.numel() != n or not w.is_contiguous() or w.get_device() != cur:
            if w.get_device() != cur:
                self._elsewhere(w, "w")
            raise ValueError(f"w: dense [{n}]")
        if q is None or scale is None:
            q, scale = self._i8_new(q, scale, T, n)
        qp, ql = self._codes(q, "q", cur, T, n)
        sp = self._floats(scale, "scale", cur, T)
        rc = self.so.mllm_i8_rms_norm(xt, xp, xl, rt, rp, rl, op, ol, wt, w.data_ptr(), eps, T, n, qp, ql, sp,
                                      self._stream_of(cur))
        if rc:
            self._check(rc, "mllm_i8_rms_norm")
        return q, scale

    def i8_silu_mul(self, gate, up, q=None, scale=None):
        """mllm_i8_silu_mul: silu(gate) * up, [T, n] each (halves of one tensor may be passed as slices) -> (q, scale)."""
        cur, gt = self._cur_raw(), self._real(gate, "gate")
        T, n = self._sizes(gate, "gate")
        gp, gl = self._at(gate, "gate", cur, T, n)
        if self._real(up, "up") != gt:
            raise TypeError("gate and up have one type")
        up_, ul = self._at(up, "up", cur, T, n)
        if q is None or scale is None:
            q, scale = self._i8_new(q, scale, T, n)
        qp, ql = self._codes(q, "q", cur, T, n)
        sp = self._floats(scale, "scale", cur, T)
        rc = self.so.mllm_i8_silu_mul(gt, gp, gl, up_, ul, T, n, qp, ql, sp, self._stream_of(cur))
        if rc:
            self._check(rc, "mllm_i8_silu_mul")
        return q, scale

    def i8_weights(self, w, scale=None):
        """An I8Weights of w [n_rows, n_cols]: float32, float16 or bfloat16 rows, quantised here (a GGUF matrix through
        dequant), or int8 rows with their own scale [n_rows]."""
        return I8Weights(self, w, scale)

    def i8_gemm_workspace(self, weights, T):
        """A workspace for i8_gemm calls of up to T tokens."""
        n = self.so.mllm_i8_gemm_workspace_size(T, weights.n_rows, weights.n_cols) if 0 <= T <= 1 << 30 else -1
        if n < 0:
            raise ValueError("i8_gemm_workspace: sizes that are not served")
        return self.torch.empty(max(n, 256), dtype=self.torch.uint8, device="cuda")

    def i8_gemm(self, weights, q, scale, bias=None, out=None, out_dtype=None, ws=None):
        """mllm_i8_gemm: q int8 [T, n_cols] (rows at multiples of 16 bytes, as the calls above make them) with scale
        float32 [T] -> out [T, n_rows] in out_dtype (None: bfloat16)."""
        cur, R = self._cur_raw(), weights.n_rows
        if weights._device != cur:
            self._made_here(cur, weights)
        T = self._sizes(q, "q")[0]
        qp, ql = self._codes(q, "q", cur, T, weights.n_cols)
        if T <= 1:
            ql = (ql + 15) // 16 * 16
        if out is None:
            out = self.torch.empty((T, R), dtype=out_dtype or self.torch.bfloat16, device="cuda")
        ot = self._real(out, "out")
        op, ol = self._at(out, "out", cur, T, R)
        if ws is None:
            ws = self.i8_gemm_workspace(weights, T)
        elif ws.get_device() != cur or not ws.is_contiguous():
            self._room(ws, cur)
        rc = self.so.mllm_i8_gemm(weights._packed, weights._scale, qp, ql, self._floats(scale, "scale", cur, T), T, R,
                                  weights.n_cols, self._floats(bias, "bias", cur, R), ot, op, ol, ws.data_ptr(), ws.nbytes,
                                  self._stream_of(cur))
        if rc:
            self._check(rc, "mllm_i8_gemm")
        return out

    def moe_prepare(self, qts, N, M, E, K, gates, ups, downs, router, renorm):
        """gates/ups/downs: per-expert raw GGUF uint8 tensors (GPU) in the
        reference's layout; router: fp32 [E][N] (GPU).  Returns a MoELayer."""
        return MoELayer(self, qts, N, M, E, K, gates, ups, downs, router, renorm)

    def moe_bucket(self, idx, E):
        """Stable bucketing of entries idx (int32 GPU, flat) over E experts."""
        torch = self.torch
        TK = idx.numel()
        max_tiles = TK // 64 + E + 1
        off = torch.empty(E + 1, dtype=torch.int32, device=idx.device)
        perm = torch.empty(TK, dtype=torch.int32, device=idx.device)
        pos_of = torch.empty(TK, dtype=torch.int32, device=idx.device)
        tiles = torch.empty(3 * max_tiles + 1, dtype=torch.int32, device=idx.device)
        self._check(self.so.mllm_moe_bucket(idx.data_ptr(), TK, E, off.data_ptr(), perm.data_ptr(), pos_of.data_ptr(),
                                            tiles.data_ptr(), self._stream()), "mllm_moe_bucket")
        n = int(tiles[3 * max_tiles].item())
        return off, perm, pos_of, (tiles[:n], tiles[max_tiles:max_tiles + n], tiles[2 * max_tiles:2 * max_tiles + n])


class MoELayer:
    """A prepared MoE layer (mllm_moe_prepare) holding its packed expert weights."""

    def __init__(self, ops, qts, N, M, E, K, gates, ups, downs, router, renorm):
        torch = ops.torch
        self.ops, self.N, self.M, self.E, self.K = ops, N, M, E, K
        sg = ops.so.mllm_sem_for(ENT_MOE_GU, qts[0]) if not (qts[0] == 39 and qts[1] == 39) else MXFP4
        su = ops.so.mllm_sem_for(ENT_MOE_GU, qts[1]) if not (qts[0] == 39 and qts[1] == 39) else MXFP4
        sd = ops.so.mllm_sem_for(ENT_MOE_DOWN, qts[2])
        self.gp = [ops.pack(sg, g, M, N) for g in gates]
        self.up = [ops.pack(su, u, M, N) for u in ups]
        self.dp = [ops.pack(sd, d, N, M) for d in downs] if sd >= 0 else [self.gp[0]] * E
        self.router = router.contiguous()
        arr = ctypes.c_void_p * E
        self.h = ops.so.mllm_moe_prepare(qts[0], qts[1], qts[2], N, M, E, K,
                                         arr(*[t.data_ptr() for t in self.gp]), arr(*[t.data_ptr() for t in self.up]),
                                         arr(*[t.data_ptr() for t in self.dp]), self.router.data_ptr(), int(renorm))
        if not self.h:
            raise RuntimeError("mllm_moe_prepare failed")
        self._ws = None

    def dense_experts(self):
        """Load-time bf16 copies of the bf16-exact expert matrices (mllm_moe_dense_experts);
        returns the bytes they take (0: no matrix of this layer qualifies)."""
        n = self.ops.so.mllm_moe_dense_experts(self.h, self.ops._stream())
        if n < 0:
            raise RuntimeError("mllm_moe_dense_experts failed: " + last_error(self.ops.so))
        return n

    def info(self):
        """mllm_moe_layer_info: bit 1 gate/up and bit 2 down on the fp16-plane GEMM,
        bit 4 the whole layer on the per-token GEMVs."""
        return self.ops.so.mllm_moe_layer_info(self.h)

    def workspace(self, T):
        n = self.ops.so.mllm_moe_workspace_size(self.h, T)
        if self._ws is None or self._ws.numel() < n:
            self._ws = self.ops.torch.empty(n, dtype=self.ops.torch.uint8, device=self.router.device)
        return self._ws

    def forward(self, x, out=None, idx=None, w=None):
        torch = self.ops.torch
        T = x.numel() // self.N
        if out is None:
            out = torch.empty((T, self.N), dtype=torch.float32, device=x.device)
        ws = self.workspace(T)
        self.ops._check(self.ops.so.mllm_moe_forward(self.h, x.data_ptr(), T, out.data_ptr(), ws.data_ptr(), ws.numel(),
                                                     idx.data_ptr() if idx is not None else None,
                                                     w.data_ptr() if w is not None else None, self.ops._stream()),
                        "mllm_moe_forward")
        return out

    def __del__(self):
        try:
            if self.h:
                self.ops.so.mllm_moe_release(self.h)
        except Exception:
            pass


class I8Weights:
    """Weights in 8-bit integers with a scale per row (mllm_i8_pack), as DeviceOps.i8_gemm takes them."""

    def __init__(self, ops, w, scale=None):
        torch, cur = ops.torch, ops._cur()
        if (w.dtype == torch.int8) != (scale is not None):
            raise ValueError("scale belongs to int8 weights")
        self.n_rows, self.n_cols = ops._sizes(w, "w")
        code, self._device = T_I8 if scale is not None else ops._real(w, "w"), cur
        wp, wl = ops._at(w, "w", cur, self.n_rows, self.n_cols)
        n = ops.so.mllm_i8_packed_size(self.n_rows, self.n_cols)
        if n < 0:
            raise ValueError("w: 1 to 131071 columns, at least one row")
        self.packed = torch.empty(n, dtype=torch.uint8, device="cuda")
        self.scale = torch.empty(self.n_rows, dtype=torch.float32, device="cuda") if scale is None else scale
        self._scale, self._packed = ops._floats(self.scale, "scale", cur, self.n_rows), self.packed.data_ptr()
        ops._check(ops.so.mllm_i8_pack(code, wp, wl, self.n_rows, self.n_cols, self._packed, self._scale,
                                       ops._raw_stream(cur)), "mllm_i8_pack")
