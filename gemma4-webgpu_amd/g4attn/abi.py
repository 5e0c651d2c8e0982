"""ctypes declarations of the C ABI in include/g4attn.h.

Loads gemma4-webgpu_amd/lib/libg4attn.so (built by gemma4-webgpu_amd/build.py).
There is no fallback: if the library is missing, loading raises.
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent.parent / "lib" / "libg4attn.so"

G4_OK = 0
G4_EINVAL = -1
G4_EHIP = -2
G4_ENOSPC = -3
G4_ENODEV = -4
G4_ERANGE = -5


class G4Error(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"g4attn status {status}: {message}")
        self.status = status
        self.message = message


# ---- Params (reference uniform layouts, src/engine.ts:526-595) -------------

class NormRopeParams(C.Structure):  # fused_per_head_norm_rope.wgsl:13
    _fields_ = [("num_heads", C.c_uint32), ("head_dim", C.c_uint32), ("eps", C.c_float),
                ("position", C.c_uint32), ("theta", C.c_float), ("apply_divisor", C.c_uint32)]


class NormParams(C.Structure):  # per_head_rms_norm_no_weight.wgsl:8
    _fields_ = [("num_heads", C.c_uint32), ("head_dim", C.c_uint32), ("eps", C.c_float), ("pad", C.c_uint32)]


class KvStoreParams(C.Structure):  # kv_cache_store.wgsl:1
    _fields_ = [("num_kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("position", C.c_uint32),
                ("max_seq_len", C.c_uint32)]


class AttnScoreParams(C.Structure):  # attn_score.wgsl:9
    _fields_ = [("num_q_heads", C.c_uint32), ("num_kv_heads", C.c_uint32), ("head_dim", C.c_uint32),
                ("seq_len", C.c_uint32), ("scale", C.c_float), ("sliding_window", C.c_uint32)]


class SoftmaxParams(C.Structure):  # softmax.wgsl:1
    _fields_ = [("num_heads", C.c_uint32), ("seq_len", C.c_uint32)]


class AttnOutputParams(C.Structure):  # attn_output.wgsl:1
    _fields_ = [("num_q_heads", C.c_uint32), ("num_kv_heads", C.c_uint32), ("head_dim", C.c_uint32),
                ("seq_len", C.c_uint32)]


class PrepParams(C.Structure):
    _fields_ = [("num_q_heads", C.c_uint32), ("num_kv_heads", C.c_uint32), ("head_dim", C.c_uint32),
                ("eps", C.c_float), ("position", C.c_uint32), ("theta", C.c_float),
                ("apply_divisor", C.c_uint32), ("slot", C.c_uint32), ("max_seq_len", C.c_uint32),
                ("store_kv", C.c_uint32)]


class PrepLayer(C.Structure):
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("q_weight", C.c_void_p),
                ("k_weight", C.c_void_p), ("rope_freqs", C.c_void_p), ("k_cache", C.c_void_p),
                ("v_cache", C.c_void_p), ("head_dim", C.c_uint32), ("theta", C.c_float),
                ("apply_divisor", C.c_uint32), ("store_kv", C.c_uint32), ("max_seq_len", C.c_uint32),
                ("reserved", C.c_uint32 * 3)]


class DecodeEntry(C.Structure):
    _fields_ = [("q", C.c_void_p), ("k_cache", C.c_void_p), ("v_cache", C.c_void_p), ("out", C.c_void_p),
                ("seq_len", C.c_uint32), ("sliding_window", C.c_uint32), ("scale", C.c_float),
                ("reserved", C.c_uint32)]


class StepEntry(C.Structure):
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("q_weight", C.c_void_p),
                ("k_weight", C.c_void_p), ("rope_freqs", C.c_void_p), ("rope_inv_freq_host", C.c_void_p),
                ("k_cache", C.c_void_p),
                ("v_cache", C.c_void_p), ("out", C.c_void_p), ("seq_len", C.c_uint32), ("position", C.c_uint32),
                ("sliding_window", C.c_uint32), ("store_kv", C.c_uint32), ("theta", C.c_float),
                ("apply_divisor", C.c_uint32), ("scale", C.c_float), ("eps", C.c_float), ("q_ready", C.c_uint32)]


class PrefillEntry(C.Structure):
    _fields_ = [("q", C.c_void_p), ("k_cache", C.c_void_p), ("v_cache", C.c_void_p), ("out", C.c_void_p),
                ("n_tokens", C.c_uint32), ("start", C.c_uint32), ("sliding_window", C.c_uint32),
                ("scale", C.c_float), ("vt_cache", C.c_void_p), ("vt_rows", C.c_uint32)]


class QkvPrepParams(C.Structure):
    _fields_ = [("num_q_heads", C.c_uint32), ("num_kv_heads", C.c_uint32), ("head_dim", C.c_uint32),
                ("position", C.c_uint32), ("slot", C.c_uint32), ("max_seq_len", C.c_uint32), ("eps", C.c_float),
                ("theta", C.c_float), ("apply_divisor", C.c_uint32), ("store_kv", C.c_uint32)]


class PromptPrepParams(C.Structure):
    _fields_ = [("num_q_heads", C.c_uint32), ("num_kv_heads", C.c_uint32), ("head_dim", C.c_uint32),
                ("n_tokens", C.c_uint32), ("start", C.c_uint32), ("eps", C.c_float), ("theta", C.c_float),
                ("apply_divisor", C.c_uint32), ("store_kv", C.c_uint32), ("max_seq_len", C.c_uint32)]


class PromptPrepEntry(C.Structure):
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("q_weight", C.c_void_p),
                ("k_weight", C.c_void_p), ("rope_freqs", C.c_void_p), ("rope_inv_freq", C.c_void_p),
                ("q_out", C.c_void_p), ("k_cache", C.c_void_p), ("v_cache", C.c_void_p), ("vt_cache", C.c_void_p),
                ("p", PromptPrepParams)]


class MatmulParams(C.Structure):  # matmul_quant.wgsl:12
    _fields_ = [("M", C.c_uint32), ("N", C.c_uint32)]


class SoftcapParams(C.Structure):  # logit_softcap.wgsl:5
    _fields_ = [("size", C.c_uint32), ("cap", C.c_float)]


class LmHeadParams(C.Structure):
    _fields_ = [("vocab", C.c_uint32), ("hidden", C.c_uint32), ("cap", C.c_float)]


class LinearSeg(C.Structure):
    _fields_ = [("weight", C.c_void_p), ("out", C.c_void_p), ("rows", C.c_uint32)]


class LinearQSeg(C.Structure):
    _fields_ = [("weight", C.c_void_p), ("meta", C.c_void_p), ("out", C.c_void_p), ("rows", C.c_uint32)]


G4_WEIGHT_F16, G4_WEIGHT_Q8, G4_WEIGHT_Q4K = 0, 1, 2


class DecodePlan(C.Structure):
    _fields_ = [("opaque", C.c_uint64 * 8)]


G4_KV_F16, G4_KV_E4M3 = 0, 1
G4_LOGITS_F32, G4_LOGITS_F16, G4_LOGITS_BF16 = 0, 1, 2
G4_LOGPROBS_MAX_TOP = 64
G4_COMMIT_MAX_CACHES = 64


class PagedCache(C.Structure):
    _fields_ = [("k_pool", C.c_void_p), ("v_pool", C.c_void_p), ("num_pages", C.c_uint32), ("page_size", C.c_uint32),
                ("num_kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("dtype", C.c_uint32), ("reserved", C.c_uint32)]


class PagedBatch(C.Structure):
    _fields_ = [("block_table", C.c_void_p), ("token_start", C.c_void_p), ("ctx_lens", C.c_void_p),
                ("positions", C.c_void_p), ("tree_mask", C.c_void_p), ("n_seqs", C.c_uint32),
                ("table_stride", C.c_uint32), ("n_tokens", C.c_uint32), ("max_tokens", C.c_uint32),
                ("mask_words", C.c_uint32), ("reserved", C.c_uint32)]


class PagedAppendParams(C.Structure):
    _fields_ = [("num_q_heads", C.c_uint32), ("eps", C.c_float), ("q_stride", C.c_uint64), ("k_stride", C.c_uint64),
                ("v_stride", C.c_uint64)]


class PagedAttnParams(C.Structure):
    _fields_ = [("num_q_heads", C.c_uint32), ("sliding_window", C.c_uint32), ("scale", C.c_float),
                ("softcap", C.c_float)]


class TokenLogprobsParams(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("vocab", C.c_uint32), ("row_stride", C.c_uint64), ("dtype", C.c_uint32),
                ("top_k", C.c_uint32), ("cap", C.c_float), ("temperature", C.c_float)]


G4_F32, G4_F16, G4_BF16, G4_E4M3 = 0, 1, 2, 3
G4_F32_SUMS = 0x100


class AddRmsNormParams(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("n", C.c_uint32), ("x_type", C.c_uint32), ("residual_type", C.c_uint32),
                ("weight_type", C.c_uint32), ("out_type", C.c_uint32), ("eps", C.c_float), ("reserved", C.c_uint32),
                ("x_stride", C.c_uint64), ("residual_stride", C.c_uint64), ("residual_out_stride", C.c_uint64),
                ("out_stride", C.c_uint64)]


class QuantizeRowsParams(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("n", C.c_uint32), ("x_type", C.c_uint32), ("reserved", C.c_uint32),
                ("x_stride", C.c_uint64), ("out_stride", C.c_uint64)]


class Lora(C.Structure):
    _fields_ = [("a", C.c_void_p), ("b", C.c_void_p), ("scales", C.c_void_p), ("n_adapters", C.c_uint32),
                ("rank", C.c_uint32), ("n", C.c_uint32), ("n_segs", C.c_uint32), ("widths", C.c_uint32 * 4),
                ("type", C.c_uint32), ("reserved", C.c_uint32)]


class LinearE4m3Params(C.Structure):
    _fields_ = [("n_tokens", C.c_uint32), ("rows", C.c_uint32), ("n", C.c_uint32), ("out_type", C.c_uint32),
                ("x_stride", C.c_uint64), ("out_stride", C.c_uint64)]


class LoraAddParams(C.Structure):
    _fields_ = [("n_tokens", C.c_uint32), ("x_type", C.c_uint32), ("out_type", C.c_uint32), ("reserved", C.c_uint32),
                ("x_stride", C.c_uint64), ("base_stride", C.c_uint64), ("out_stride", C.c_uint64)]


_P = C.c_void_p
_U32 = C.c_uint32
_SZ = C.c_size_t
_INT = C.c_int

# name -> argtypes (restype is int status for all but the two string getters)
SIGNATURES: dict[str, list] = {
    "g4_device_count": [C.POINTER(C.c_int)],
    "g4_set_device": [_INT],
    "g4_stream_create": [C.POINTER(C.c_void_p)],
    "g4_stream_destroy": [_P],
    "g4_stream_synchronize": [_P],
    "g4_malloc": [C.POINTER(C.c_void_p), _SZ],
    "g4_free": [_P],
    "g4_upload": [_P, _SZ, _P, _SZ, _P],
    "g4_download": [_P, _P, _SZ, _SZ, _P],
    "g4_readback_begin": [_P, _SZ, _SZ, _P, C.POINTER(_P)],
    "g4_readback_finish": [_P, _P],
    "g4_query_set_create": [_U32, C.POINTER(_P)],
    "g4_query_begin_pass": [_P, _U32],
    "g4_query_end_pass": [],
    "g4_query_write": [_P, _U32, _P],
    "g4_query_resolve": [_P, _U32, _U32, C.POINTER(C.c_double)],
    "g4_query_set_destroy": [_P],
    "g4_zero": [_P, _SZ, _P],
    "g4_fused_per_head_norm_rope": [_P, _P, _P, NormRopeParams, _P],
    "g4_per_head_rms_norm_no_weight": [_P, NormParams, _P],
    "g4_kv_cache_store": [_P, _P, _P, _P, KvStoreParams, _P],
    "g4_attn_score": [_P, _P, _P, AttnScoreParams, _P],
    "g4_softmax": [_P, SoftmaxParams, _P],
    "g4_attn_output": [_P, _P, _P, AttnOutputParams, _P],
    "g4_attn_prep": [_P, _P, _P, _P, _P, _P, _P, _P, PrepParams, _P],
    "g4_attn_prep_many": [_P, _U32, _U32, _U32, C.c_float, _U32, _U32, _P],
    "g4_attn_decode_workspace_size": [_U32, _U32, _U32, _U32, C.POINTER(C.c_size_t)],
    "g4_attn_decode": [_P, _P, _P, _P, AttnScoreParams, _P, _SZ, _P],
    "g4_attn_decode_noalloc": [_P, _P, _P, _P, AttnScoreParams, _P],
    "g4_attn_decode_many_workspace_size": [_U32, _U32, _U32, _U32, C.c_uint64, C.POINTER(C.c_size_t)],
    "g4_attn_decode_many_prepare": [C.POINTER(DecodeEntry), _U32, _U32, _U32, _U32, _P, _SZ,
                                    C.POINTER(DecodePlan), _P],
    "g4_attn_decode_many_run": [C.POINTER(DecodePlan), _P],
    "g4_attn_decode_many_run_split": [C.POINTER(DecodePlan), _P],
    "g4_attn_decode_many_run_merge": [C.POINTER(DecodePlan), _P],
    "g4_attn_decode_many": [C.POINTER(DecodeEntry), _U32, _U32, _U32, _U32, _P, _SZ, _P],
    "g4_attn_step_workspace_size": [_U32, _U32, _U32, _U32, C.POINTER(C.c_size_t)],
    "g4_attn_step_prepare": [C.POINTER(StepEntry), _U32, _U32, _U32, _U32, _P, _SZ, C.POINTER(DecodePlan), _P],
    "g4_attn_step_layers_workspace_size": [_U32, _U32, _U32, _U32, _U32, C.POINTER(C.c_size_t)],
    "g4_attn_step_prepare_layers": [C.POINTER(StepEntry), _U32, _U32, _U32, _U32, _U32, _P, _SZ,
                                    C.POINTER(DecodePlan), _P],
    "g4_rope_inv_freq": [C.c_float, _U32, _U32, _P, _P, _P],
    "g4_rope_inv_freq_host": [C.c_float, _U32, _U32, _P, _P],
    "g4_attn_step_run": [C.POINTER(DecodePlan), _P],
    "g4_attn_step_advance": [C.POINTER(DecodePlan), C.c_uint32],
    "g4_attn_step_run_attention": [C.POINTER(DecodePlan), _P],
    "g4_attn_step_run_merge": [C.POINTER(DecodePlan), _P],
    "g4_attn_step_run_out": [C.POINTER(DecodePlan), C.POINTER(LinearSeg), _U32, _P],
    "g4_attn_step_run_attention_timed": [C.POINTER(DecodePlan), _P, _P, _P],
    "g4_attn_step_run_attention_pair": [C.POINTER(DecodePlan), C.POINTER(DecodePlan), _P],
    "g4_attn_step_run_attention_pair_timed": [C.POINTER(DecodePlan), C.POINTER(DecodePlan), _P, _P, _P],
    "g4_attn_step_run_pair": [C.POINTER(DecodePlan), C.POINTER(DecodePlan), _P],
    "g4_attn_step": [C.POINTER(StepEntry), _U32, _U32, _U32, _U32, _P, _SZ, _P],
    "g4_attn_prefill_workspace_size": [C.POINTER(PrefillEntry), _U32, _U32, _U32, _U32, C.POINTER(C.c_size_t)],
    "g4_attn_prefill_prepare": [C.POINTER(PrefillEntry), _U32, _U32, _U32, _U32, _P, _SZ, C.POINTER(DecodePlan),
                                _P],
    "g4_attn_prefill_run": [C.POINTER(DecodePlan), _P],
    "g4_attn_prefill_run_timed": [C.POINTER(DecodePlan), _P, _P, _P],
    "g4_attn_prefill": [C.POINTER(PrefillEntry), _U32, _U32, _U32, _U32, _P, _SZ, _P],
    "g4_attn_prompt_prep": [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, PromptPrepParams, _P],
    "g4_attn_prompt_prep_vt": [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, PromptPrepParams, _P],
    "g4_attn_prompt_prep_many": [C.POINTER(PromptPrepEntry), C.c_uint32, _P],
    "g4_matmul_quant_f16": [_P, _P, _P, MatmulParams, _P],
    "g4_linear_f16": [_P, _U32, C.POINTER(LinearSeg), _U32, _P],
    "g4_read_ceiling": [_P, _SZ, _P, _P, _P, _P],
    "g4_matmul_q8": [_P, _P, _P, _P, MatmulParams, _P],
    "g4_matmul_q4k": [_P, _P, _P, _P, MatmulParams, _P],
    "g4_linear_quant": [_P, _U32, _U32, C.POINTER(LinearQSeg), _U32, _P],
    "g4_linear_qkv_prep_workspace_size": [_U32, _U32, C.POINTER(C.c_size_t)],
    "g4_linear_qkv_prep": [_P, _U32, _U32, C.POINTER(LinearQSeg), _U32, _P, _P, _P, _P, _P, _P, QkvPrepParams, _P, _P],
    "g4_logit_softcap": [_P, SoftcapParams, _P],
    "g4_argmax": [_P, _P, _U32, _P],
    "g4_lm_head_workspace_size": [LmHeadParams, C.POINTER(C.c_size_t)],
    "g4_lm_head_argmax": [_P, _P, _P, _P, _P, _SZ, LmHeadParams, _P],
    "g4_lm_head_argmax_timed": [_P, _P, _P, _P, _P, _SZ, LmHeadParams, _P, _P, _P],
    "g4_paged_append": [C.POINTER(PagedCache), C.POINTER(PagedBatch), _P, _P, _P, _P, _P, _P, _P,
                        C.POINTER(PagedAppendParams), _P],
    "g4_paged_attn_workspace_size": [C.POINTER(PagedCache), C.POINTER(PagedBatch), _U32, C.POINTER(C.c_size_t)],
    "g4_paged_attn": [C.POINTER(PagedCache), C.POINTER(PagedBatch), _P, _P, C.POINTER(PagedAttnParams), _P, _SZ, _P],
    "g4_paged_commit": [C.POINTER(PagedCache), _U32, C.POINTER(PagedBatch), _P, _U32, _P, _P, _P],
    "g4_token_logprobs_workspace_size": [C.POINTER(TokenLogprobsParams), C.POINTER(C.c_size_t)],
    "g4_token_logprobs": [_P, _P, _P, _P, _P, _P, C.POINTER(TokenLogprobsParams), _P, _SZ, _P],
    "g4_add_rms_norm": [_P, _P, _P, _P, _P, _P, _P, C.POINTER(AddRmsNormParams), _P],
    "g4_quantize_rows": [_P, _P, _P, C.POINTER(QuantizeRowsParams), _P],
    "g4_linear_e4m3_workspace_size": [C.POINTER(LinearE4m3Params), C.POINTER(Lora), C.POINTER(C.c_size_t)],
    "g4_linear_e4m3": [_P, _P, _P, _P, C.POINTER(Lora), _P, _P, C.POINTER(LinearE4m3Params), _P, _SZ, _P],
    "g4_lora_workspace_size": [C.POINTER(Lora), _U32, C.POINTER(C.c_size_t)],
    "g4_lora_add": [C.POINTER(Lora), _P, _P, _P, _P, _P, C.POINTER(LoraAddParams), _P, _SZ, _P],
}
STRING_FUNCS = ("g4_last_error", "g4_version")

_lib: C.CDLL | None = None


def load() -> C.CDLL:
    """Load libg4attn.so once; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    path = Path(os.environ.get("G4ATTN_LIB", LIB_PATH))
    if not path.exists():
        raise FileNotFoundError(f"{path} not built: run `python gemma4-webgpu_amd/build.py`")
    lib = C.CDLL(str(path))
    for name in STRING_FUNCS:
        f = getattr(lib, name)
        f.restype = C.c_char_p
        f.argtypes = []
    for name, args in SIGNATURES.items():
        f = getattr(lib, name)
        f.restype = C.c_int
        f.argtypes = args
    _lib = lib
    return lib


def check(status: int) -> None:
    if status != G4_OK:
        msg = load().g4_last_error().decode(errors="replace")
        raise G4Error(status, msg)


def call(name: str, *args) -> None:
    check(getattr(load(), name)(*args))
