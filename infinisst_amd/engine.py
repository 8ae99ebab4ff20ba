"""ctypes binding of libinfinisst_hip.so (include/infinisst_hip.h) -- the only compute path of this package.

There is no CPU fallback: if the HIP library is missing or no GPU is visible, construction fails loudly.
PyTorch is used here for plumbing only (device tensors handed over as raw pointers, the current HIP stream).
"""
from __future__ import annotations

import ctypes as C
import itertools
import os
import time
from typing import Dict, Optional, Sequence

import numpy as np
import torch

from . import rope
from .config import GenConfig, ModelConfig

_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libinfinisst_hip.so")
_lib = None

ISST_MAX_CONV, ISST_MAX_SHRINK, ISST_MAX_EOS = 8, 4, 8

EPI = {"none": 0, "bias": 1, "bias_gelu": 2, "res": 3, "bias_res": 4, "swiglu": 5, "f32": 6, "swiglu8": 8}


class IsstError(RuntimeError):
    pass


class _Config(C.Structure):
    _fields_ = [
        ("n_conv", C.c_int), ("conv_dim", C.c_int * ISST_MAX_CONV), ("conv_k", C.c_int * ISST_MAX_CONV),
        ("conv_stride", C.c_int * ISST_MAX_CONV), ("conv_bias", C.c_int),
        ("enc_dim", C.c_int), ("enc_layers", C.c_int), ("enc_heads", C.c_int), ("enc_ffn", C.c_int),
        ("enc_ln_eps", C.c_float), ("block_size", C.c_int), ("max_cache_size", C.c_int),
        ("enc_rope_round_each", C.c_int),
        ("n_shrink", C.c_int), ("shrink_dim", C.c_int * ISST_MAX_SHRINK), ("shrink_k", C.c_int * ISST_MAX_SHRINK),
        ("shrink_stride", C.c_int * ISST_MAX_SHRINK),
        ("llm_dim", C.c_int), ("llm_layers", C.c_int), ("llm_heads", C.c_int), ("llm_kv_heads", C.c_int),
        ("llm_ffn", C.c_int), ("vocab", C.c_int), ("rms_eps", C.c_float),
        ("user_id", C.c_int), ("assistant_id", C.c_int), ("start_header_id", C.c_int),
        ("n_eos", C.c_int), ("eos_ids", C.c_int * ISST_MAX_EOS),
        ("max_streams", C.c_int), ("max_multiplier", C.c_int), ("max_prompt_len", C.c_int),
        ("max_new_tokens", C.c_int), ("max_llm_cache_size", C.c_int), ("max_system_prompt", C.c_int),
        ("debug_taps", C.c_int), ("max_beams", C.c_int), ("enc_abs_pos", C.c_int),
    ]


class _GenParams(C.Structure):
    _fields_ = [
        ("multiplier", C.c_int), ("max_new_tokens", C.c_int), ("no_repeat_ngram_size", C.c_int),
        ("encoder_no_repeat_ngram_size", C.c_int), ("repetition_penalty", C.c_float),
        ("suppress_tokens", C.POINTER(C.c_int)), ("n_suppress", C.c_int), ("system_prompt_size", C.c_int),
        ("num_beams", C.c_int), ("length_penalty", C.c_float), ("pcm_on_device", C.c_int),
        ("do_sample", C.c_int), ("temperature", C.c_float), ("top_k", C.c_int), ("top_p", C.c_float), ("epsilon_cutoff", C.c_float),
        ("seed", C.c_ulonglong),
    ]


class _StreamInfo(C.Structure):
    _fields_ = [("llm_cache_len", C.c_int), ("llm_sys_len", C.c_int), ("enc_n_steps", C.c_int),
                ("enc_cache_len", C.c_int), ("chunks", C.c_int)]


class _PrefixAttn(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("q", "k_prefix", "v_prefix", "k_tail", "v_tail", "tail_lens", "row_starts", "out")]
                + [(n, C.c_int64) for n in ("q_row", "q_head", "out_row", "out_head", "kp_head", "kp_key", "vp_head", "vp_key",
                                            "kt_seq", "kt_head", "kt_key", "vt_seq", "vt_head", "vt_key")]
                + [(n, C.c_int) for n in ("rows", "seqs", "max_rows", "heads", "kv_heads", "head_dim", "prefix_len", "tail_cap")] + [("scale", C.c_float)])


# every symbol include/infinisst_hip.h declares
EXPORTS = [
    "isst_create", "isst_destroy", "isst_last_error", "isst_load_weight", "isst_set_rope_tables", "isst_set_enc_position_table",
    "isst_finalize_weights", "isst_stream_open", "isst_stream_reset", "isst_stream_close", "isst_stream_info_get",
    "isst_stream_import_llm_kv", "isst_stream_import_enc_kv", "isst_stream_import_audio_history",
    "isst_debug_beam_trace_begin", "isst_debug_beam_trace_step", "isst_debug_beam_trace_end",
    "isst_op_attn_combine", "isst_op_gemm_attn_merge", "isst_op_splice_map", "isst_op_embed_splice", "isst_op_enc_attention", "isst_op_llm_attention",
    "isst_generate", "isst_kv_evict", "isst_encode_speech", "isst_debug_tap", "isst_debug_read_kv", "isst_profile_begin", "isst_profile_begin_rows", "isst_profile_end", "isst_op_pack_weight", "isst_op_pack_gateup8",
    "isst_op_packed_elems", "isst_op_gemm", "isst_op_gemm_splitk_rmsnorm", "isst_op_gemm_splitk_fused", "isst_op_gemm_splitk_plain", "isst_op_gemm_norm_ssq", "isst_op_gemm_splitk_layernorm", "isst_op_set_gemm_tuning", "isst_op_set_attn_tuning", "isst_op_set_reduce_tuning", "isst_op_topk_rows", "isst_op_layernorm", "isst_op_rmsnorm", "isst_op_conv0", "isst_op_sample", "isst_op_warp", "isst_op_warp_sample", "isst_op_sample_uniform", "isst_op_multinomial_wor",
    "isst_op_prefix_attention", "isst_op_prefix_attention_workspace", "isst_op_gemm_lora", "isst_op_gemm_lora_workspace", "isst_op_verify_drafts", "isst_op_verify_drafts_workspace",
]


def load_library(path: Optional[str] = None):
    """dlopen the HIP library; raises if it has not been built (python __graft_entry__.py / make -C csrc)."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = path or _LIB_PATH
    if not os.path.exists(p):
        raise IsstError(f"{p} not found: build it with `make -C infinisst_amd/csrc` (no CPU fallback exists)")
    lib = C.CDLL(p)
    lib.isst_last_error.restype = C.c_char_p
    lib.isst_last_error.argtypes = [C.c_void_p]
    lib.isst_destroy.restype = None
    lib.isst_destroy.argtypes = [C.c_void_p]
    lib.isst_op_packed_elems.restype = C.c_int64
    lib.isst_create.argtypes = [C.POINTER(_Config), C.POINTER(C.c_void_p)]
    lib.isst_load_weight.argtypes = [C.c_void_p, C.c_char_p, C.c_void_p, C.c_int, C.POINTER(C.c_int64), C.c_int]
    lib.isst_set_rope_tables.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int]
    lib.isst_set_enc_position_table.argtypes = [C.c_void_p, C.c_void_p, C.c_int]
    lib.isst_finalize_weights.argtypes = [C.c_void_p]
    lib.isst_stream_open.argtypes = [C.c_void_p, C.POINTER(C.c_int)]
    lib.isst_stream_reset.argtypes = [C.c_void_p, C.c_int]
    lib.isst_stream_close.argtypes = [C.c_void_p, C.c_int]
    lib.isst_stream_info_get.argtypes = [C.c_void_p, C.c_int, C.POINTER(_StreamInfo)]
    lib.isst_kv_evict.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int]
    lib.isst_stream_import_llm_kv.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int]
    lib.isst_stream_import_enc_kv.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int]
    lib.isst_stream_import_audio_history.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_int]
    lib.isst_debug_beam_trace_begin.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int]
    lib.isst_debug_beam_trace_step.argtypes = [C.c_void_p, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_int), C.c_void_p, C.c_void_p, C.c_void_p, C.c_int]
    lib.isst_debug_beam_trace_end.argtypes = [C.c_void_p, C.POINTER(C.c_int)]
    lib.isst_op_attn_combine.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p]
    lib.isst_op_gemm_attn_merge.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_void_p]
    lib.isst_op_splice_map.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.POINTER(C.c_int)]
    lib.isst_op_embed_splice.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p]
    lib.isst_op_enc_attention.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p,
                                          C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p]
    lib.isst_op_llm_attention.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int,
                                          C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]
    lib.isst_generate.argtypes = [C.c_void_p, C.POINTER(_GenParams), C.c_int, C.POINTER(C.c_int),
                                  C.POINTER(C.c_void_p), C.c_int, C.POINTER(C.c_void_p), C.POINTER(C.c_int),
                                  C.POINTER(C.c_void_p), C.POINTER(C.c_int), C.POINTER(C.c_void_p), C.POINTER(C.c_int),
                                  C.POINTER(C.c_void_p), C.POINTER(C.c_int), C.c_void_p, C.c_void_p]
    lib.isst_encode_speech.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int, C.c_void_p,
                                       C.POINTER(C.c_int), C.c_void_p]
    lib.isst_debug_tap.argtypes = [C.c_void_p, C.c_char_p, C.c_void_p, C.c_int64, C.POINTER(C.c_int64)]
    lib.isst_debug_read_kv.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p]
    lib.isst_profile_begin.argtypes = [C.c_void_p]
    lib.isst_profile_begin_rows.argtypes = [C.c_void_p, C.c_int, C.c_int]
    lib.isst_profile_end.argtypes = [C.c_void_p, C.c_void_p, C.POINTER(C.c_double), C.POINTER(C.c_int64)]
    lib.isst_op_pack_weight.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p]
    lib.isst_op_packed_elems.argtypes = [C.c_int, C.c_int]
    lib.isst_op_pack_gateup8.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p]
    lib.isst_op_gemm.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p,
                                 C.c_int64, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_float, C.c_void_p]
    lib.isst_op_gemm_splitk_rmsnorm.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                                C.c_int, C.c_int, C.c_int, C.c_int, C.c_float, C.c_void_p]
    lib.isst_op_gemm_splitk_layernorm.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                                  C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_float, C.c_void_p]
    lib.isst_op_set_gemm_tuning.argtypes = [C.c_int, C.c_int]
    lib.isst_op_set_attn_tuning.argtypes = [C.c_int]
    lib.isst_op_set_reduce_tuning.argtypes = [C.c_int, C.c_int]
    lib.isst_op_layernorm.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_float,
                                      C.c_int, C.c_void_p]
    lib.isst_op_rmsnorm.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_float, C.c_void_p]
    lib.isst_op_conv0.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int,
                                  C.c_int, C.c_int, C.c_int, C.c_void_p]
    lib.isst_op_warp_sample.argtypes = [C.c_void_p, C.c_int, C.c_float, C.c_int, C.c_float, C.c_float, C.c_double, C.POINTER(C.c_int)]
    lib.isst_op_topk_rows.argtypes = [C.c_void_p, C.c_long, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
    lib.isst_op_sample_uniform.argtypes = [C.c_ulonglong, C.c_int, C.c_int, C.c_int]
    lib.isst_op_sample_uniform.restype = C.c_double
    lib.isst_op_sample.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_int,
                                   C.c_float, C.c_int, C.c_int, C.c_void_p, C.c_void_p]
    lib.isst_op_prefix_attention_workspace.argtypes = [C.POINTER(_PrefixAttn)]
    lib.isst_op_prefix_attention_workspace.restype = C.c_int64
    lib.isst_op_prefix_attention.argtypes = [C.POINTER(_PrefixAttn), C.c_void_p, C.c_int64, C.c_void_p]
    lib.isst_op_gemm_lora_workspace.argtypes = [C.c_int] * 5
    lib.isst_op_gemm_lora_workspace.restype = C.c_int64
    lib.isst_op_gemm_lora.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_int64,
                                      C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_int64, C.c_void_p]
    lib.isst_op_verify_drafts_workspace.argtypes = [C.c_int] * 3
    lib.isst_op_verify_drafts_workspace.restype = C.c_int64
    lib.isst_op_verify_drafts.argtypes = [C.c_void_p, C.c_int64, C.c_int64, C.c_void_p, C.c_int64, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                          C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
    if path is None:
        _lib = lib
    return lib


def _stream_ptr() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else C.c_void_p(t.data_ptr())


def make_c_config(cfg: ModelConfig, max_streams: int, max_multiplier: int, max_prompt_len: int, max_new_tokens: int,
                  max_llm_cache_size: int, max_system_prompt: int, debug_taps: bool, max_beams: int = 1) -> _Config:
    c = _Config()
    c.n_conv = len(cfg.conv_layers)
    for i, (d, k, s) in enumerate(cfg.conv_layers):
        c.conv_dim[i], c.conv_k[i], c.conv_stride[i] = d, k, s
    c.conv_bias = int(cfg.conv_bias)
    c.enc_dim, c.enc_layers, c.enc_heads, c.enc_ffn = cfg.enc_dim, cfg.enc_layers, cfg.enc_heads, cfg.enc_ffn
    c.enc_ln_eps, c.block_size, c.max_cache_size = cfg.enc_ln_eps, cfg.block_size, cfg.max_cache_size
    c.enc_rope_round_each = int(cfg.enc_rope_mode == "bf16")
    c.n_shrink = len(cfg.shrink_layers)
    for i, (d, k, s) in enumerate(cfg.shrink_layers):
        c.shrink_dim[i], c.shrink_k[i], c.shrink_stride[i] = d, k, s
    if cfg.llm_head_dim != 128:
        raise IsstError("llm_head_dim must be 128")
    c.llm_dim, c.llm_layers, c.llm_heads, c.llm_kv_heads = cfg.llm_dim, cfg.llm_layers, cfg.llm_heads, cfg.llm_kv_heads
    c.llm_ffn, c.vocab, c.rms_eps = cfg.llm_ffn, cfg.vocab, cfg.rms_eps
    c.user_id, c.assistant_id, c.start_header_id = cfg.user_id, cfg.assistant_id, cfg.start_header_id
    c.n_eos = len(cfg.eos_ids)
    for i, e in enumerate(cfg.eos_ids):
        c.eos_ids[i] = e
    c.max_streams, c.max_multiplier, c.max_prompt_len = max_streams, max_multiplier, max_prompt_len
    c.max_new_tokens, c.max_llm_cache_size, c.max_system_prompt = max_new_tokens, max_llm_cache_size, max_system_prompt
    c.debug_taps = int(debug_taps)
    c.max_beams = max_beams
    c.enc_abs_pos = int(not cfg.enc_rope)
    return c


def _pack_int32(seqs, n: int):
    """n int32 sequences (lists, arrays or None) -> (owner of the memory, c_void_p[n] pointing into it or NULL, c_int[n] lengths)."""
    if len(seqs) != n:
        raise IsstError(f"{len(seqs)} sequences for {n} streams")
    lens = [0 if s is None else len(s) for s in seqs]
    total = sum(lens)
    if total == 0:
        return None, (C.c_void_p * n)(), (C.c_int * n)(*lens)
    live = [s for s, l in zip(seqs, lens) if l]
    if all(isinstance(s, np.ndarray) for s in live):
        flat = np.concatenate(live).astype(np.int32, copy=False)
    else:
        flat = np.fromiter(itertools.chain.from_iterable(live), dtype=np.int32, count=total)
    flat = np.ascontiguousarray(flat)
    base = flat.ctypes.data
    ptrs, off = [], 0
    for l in lens:
        ptrs.append(base + 4 * off if l else None)
        off += l
    return flat, (C.c_void_p * n)(*ptrs), (C.c_int * n)(*lens)


class Engine:
    """Owns one library handle: device weights + per-stream KV state on the current CUDA(HIP) device."""

    def __init__(self, cfg: ModelConfig, max_streams: int = 1, max_multiplier: int = 1, max_prompt_len: int = 128,
                 max_new_tokens: int = 40, max_llm_cache_size: int = 1000, max_system_prompt: int = 128,
                 debug_taps: bool = False, max_beams: int = 1):
        if not torch.cuda.is_available():
            raise IsstError("no GPU visible: the InfiniSST hot path has no CPU implementation in this package")
        self.lib = load_library()
        self.cfg = cfg
        self.c_cfg = make_c_config(cfg, max_streams, max_multiplier, max_prompt_len, max_new_tokens,
                                   max_llm_cache_size, max_system_prompt, debug_taps, max_beams)
        self.max_new_tokens = max_new_tokens
        self.last_call_seconds = 0.0
        r64 = lambda x: (x + 63) // 64 * 64
        # rows the library wants from isst_set_rope_tables (engine_core.hip isst_create: sys_cap + ring_cap, enc_cap)
        self._llm_rope_rows = r64(max_system_prompt) + r64(max_llm_cache_size + max_prompt_len + max_new_tokens + 8)
        self._enc_rope_rows = r64(cfg.max_cache_size + cfg.block_size * max_multiplier)
        self.h = C.c_void_p()
        rc = self.lib.isst_create(C.byref(self.c_cfg), C.byref(self.h))
        if rc != 0:
            raise IsstError(f"isst_create failed ({rc}): {self.lib.isst_last_error(None).decode()}")

    # ---------------------------------------------------------------- errors / lifetime
    def _check(self, rc: int, what: str):
        if rc != 0:
            raise IsstError(f"{what} failed ({rc}): {self.lib.isst_last_error(self.h).decode()}")

    def close(self):
        if getattr(self, "h", None) is not None and self.h.value:
            self.lib.isst_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---------------------------------------------------------------- weights
    def load_checkpoint(self, path: str):
        """Reference `pytorch_model.bin` (agents/infinisst.py:179-180) -> device weights; returns the skipped keys."""
        from .checkpoint import load_checkpoint
        weights, inv_freq, skipped = load_checkpoint(self.cfg, path)
        self.load_weights(weights, enc_inv_freq=inv_freq)
        return skipped

    def load_weights(self, weights: Dict[str, torch.Tensor], strict: bool = True, enc_inv_freq=None):
        """`weights`: reference checkpoint keys -> bf16 tensors (CPU or GPU).  Unknown keys raise if strict."""
        for name, t in weights.items():
            if t.dtype != torch.bfloat16:
                raise IsstError(f"{name}: expected bfloat16, got {t.dtype}")
            t = t.contiguous()
            shape = (C.c_int64 * t.dim())(*t.shape)
            rc = self.lib.isst_load_weight(self.h, name.encode(), C.c_void_p(t.data_ptr()), t.dim(), shape, int(t.is_cuda))
            if rc == -5 and not strict:
                continue
            self._check(rc, f"isst_load_weight({name})")
        rows_e, rows_l = max(1024, self._enc_rope_rows), max(1 << 14, self._llm_rope_rows)
        ec, es = rope.encoder_tables(self.cfg, rows_e, enc_inv_freq)
        lc, ls = rope.llm_tables(self.cfg, rows_l)
        self._check(self.lib.isst_set_rope_tables(self.h, C.c_void_p(ec.data_ptr()), C.c_void_p(es.data_ptr()), rows_e,
                                                  C.c_void_p(lc.data_ptr()), C.c_void_p(ls.data_ptr()), rows_l),
                    "isst_set_rope_tables")
        if not self.cfg.enc_rope:
            table = rope.encoder_position_table(self.cfg)
            self._check(self.lib.isst_set_enc_position_table(self.h, C.c_void_p(table.data_ptr()), table.shape[0]), "isst_set_enc_position_table")
        self._check(self.lib.isst_finalize_weights(self.h), "isst_finalize_weights")
        torch.cuda.synchronize()

    # ---------------------------------------------------------------- streams
    def open_stream(self) -> int:
        sid = C.c_int(-1)
        self._check(self.lib.isst_stream_open(self.h, C.byref(sid)), "isst_stream_open")
        return sid.value

    def reset_stream(self, sid: int):
        self._check(self.lib.isst_stream_reset(self.h, sid), "isst_stream_reset")

    def close_stream(self, sid: int):
        self._check(self.lib.isst_stream_close(self.h, sid), "isst_stream_close")

    def stream_info(self, sid: int) -> dict:
        info = _StreamInfo()
        self._check(self.lib.isst_stream_info_get(self.h, sid, C.byref(info)), "isst_stream_info_get")
        return {k: getattr(info, k) for k, _ in _StreamInfo._fields_}

    def stream_cache_lens(self, sids: Sequence[int]) -> list:
        """llm_cache_len of several streams (what the agent reads as past_key_values[0][0].size(2), agents/infinisst.py:337)."""
        info = _StreamInfo()
        ref = C.byref(info)
        out = []
        for sid in sids:
            self._check(self.lib.isst_stream_info_get(self.h, sid, ref), "isst_stream_info_get")
            out.append(info.llm_cache_len)
        return out

    def kv_evict(self, sid: int, new_cache_size: int, keep_prefix: int):
        self._check(self.lib.isst_kv_evict(self.h, sid, new_cache_size, keep_prefix), "isst_kv_evict")

    # ---------------------------------------------------------------- state import (resume / steady-state set-up)
    def import_llm_kv(self, sid: int, kv, sys_len: int, ring_start: int = 0):
        """`kv`: past_key_values as a list over layers of (K, V), each (1, kv_heads, T, 128) bf16 with UNROTATED keys
        (the reference's patched cache, model/patches/patch_llm.py:280-284); the first `sys_len` entries become the pinned prefix."""
        if len(kv) != self.cfg.llm_layers:
            raise IsstError(f"{len(kv)} layers given, the model has {self.cfg.llm_layers}")
        for layer, (k, v) in enumerate(kv):
            k = k.detach().to("cpu", torch.bfloat16).reshape(self.cfg.llm_kv_heads, -1, 128).contiguous()
            v = v.detach().to("cpu", torch.bfloat16).reshape(self.cfg.llm_kv_heads, -1, 128).contiguous()
            self._check(self.lib.isst_stream_import_llm_kv(self.h, sid, layer, C.c_void_p(k.data_ptr()), C.c_void_p(v.data_ptr()), k.shape[1],
                                                           sys_len, ring_start), "isst_stream_import_llm_kv")

    def import_speech_cache(self, sid: int, layers, n_steps: int, audio_tail=None, ring_start: int = 0):
        """`layers`: per encoder layer (K, V), each (heads, T, 64) bf16 with unrotated keys (= speech_cache.layers[i].k / .v, reference
        model/speech_encoder.py:80-97); `n_steps` = speech_cache.n_steps; `audio_tail`: the last 399 samples of speech_cache.src."""
        if len(layers) != self.cfg.enc_layers:
            raise IsstError(f"{len(layers)} layers given, the encoder has {self.cfg.enc_layers}")
        for layer, (k, v) in enumerate(layers):
            k = k.detach().to("cpu", torch.bfloat16).reshape(self.cfg.enc_heads, -1, 64).contiguous()
            v = v.detach().to("cpu", torch.bfloat16).reshape(self.cfg.enc_heads, -1, 64).contiguous()
            self._check(self.lib.isst_stream_import_enc_kv(self.h, sid, layer, C.c_void_p(k.data_ptr()), C.c_void_p(v.data_ptr()), k.shape[1],
                                                           n_steps, ring_start), "isst_stream_import_enc_kv")
        if audio_tail is not None:
            a = torch.as_tensor(audio_tail).detach().to("cpu", torch.bfloat16).reshape(-1).contiguous()
            self._check(self.lib.isst_stream_import_audio_history(self.h, sid, C.c_void_p(a.data_ptr()), a.numel()), "isst_stream_import_audio_history")

    # ---------------------------------------------------------------- beam-search test aid
    def beam_trace_begin(self, num_beams: int, forced_tokens=None, forced_parents=None):
        ft = np.ascontiguousarray(np.asarray(forced_tokens if forced_tokens is not None else [], dtype=np.int32).reshape(-1))
        fp = np.ascontiguousarray(np.asarray(forced_parents if forced_parents is not None else [], dtype=np.int32).reshape(-1))
        steps = ft.size // num_beams
        self._check(self.lib.isst_debug_beam_trace_begin(self.h, num_beams, ft.ctypes.data if steps else None, fp.ctypes.data if steps else None, steps),
                    "isst_debug_beam_trace_begin")

    def beam_trace_end(self):
        """-> list over steps of (top_val [rows][n_keep], top_idx [rows][n_keep], beam_scores [rows])."""
        n = C.c_int(0)
        out = []
        step = 0
        while True:
            rows, keep = C.c_int(0), C.c_int(0)
            if self.lib.isst_debug_beam_trace_step(self.h, step, C.byref(rows), C.byref(keep), None, None, None, 0) != 0:
                break
            val = np.zeros((rows.value, keep.value), dtype=np.float32)
            idx = np.zeros((rows.value, keep.value), dtype=np.int32)
            sc = np.zeros(rows.value, dtype=np.float32)
            self._check(self.lib.isst_debug_beam_trace_step(self.h, step, C.byref(rows), C.byref(keep), val.ctypes.data, idx.ctypes.data,
                                                            sc.ctypes.data, val.size), "isst_debug_beam_trace_step")
            out.append((val, idx, sc))
            step += 1
        self._check(self.lib.isst_debug_beam_trace_end(self.h, C.byref(n)), "isst_debug_beam_trace_end")
        return out

    # ---------------------------------------------------------------- hot path
    def generate(self, gen: GenConfig, stream_ids: Sequence[int], pcm: Sequence[np.ndarray],
                 prompt_ids: Sequence[Sequence[int]], prev_target_ids: Sequence[Sequence[int]],
                 system_prompt_size: int = 0, forced_tokens: Optional[Sequence[Optional[Sequence[int]]]] = None,
                 return_logits: bool = False):
        """model.generate(...) of reference agents/infinisst.py:307-332 for len(stream_ids) streams.
        `pcm`: one fp32 waveform segment per stream -- numpy arrays (host; the library uploads them, reference :222) or, all of them,
        contiguous fp32 CUDA tensors (audio already resident in HBM: isst_gen_params.pcm_on_device).
        Returns (list of generated id lists, logits or None)."""
        n = len(stream_ids)
        on_device = len(pcm) > 0 and all(isinstance(x, torch.Tensor) and x.is_cuda for x in pcm)
        if on_device:
            if any(x.dtype != torch.float32 or not x.is_contiguous() or x.dim() != 1 for x in pcm):
                raise IsstError("device audio must be contiguous 1-D fp32 tensors")
            pcm = list(pcm)
        else:
            pcm = [np.ascontiguousarray(x, dtype=np.float32) for x in pcm]
        n_samples = int(pcm[0].shape[0])
        if any(tuple(x.shape) != (n_samples,) for x in pcm):
            raise IsstError("all streams of one call must bring the same number of samples")
        p = _GenParams()
        p.pcm_on_device = int(on_device)
        p.multiplier, p.max_new_tokens = gen.latency_multiplier, gen.max_new_tokens
        p.no_repeat_ngram_size = p.encoder_no_repeat_ngram_size = gen.no_repeat_ngram_size
        p.repetition_penalty = gen.repetition_penalty
        sup = np.asarray(gen.suppress_tokens, dtype=np.int32)
        p.suppress_tokens = sup.ctypes.data_as(C.POINTER(C.c_int)) if sup.size else None
        p.n_suppress = int(sup.size)
        p.system_prompt_size = system_prompt_size
        p.num_beams = gen.beam
        p.length_penalty = 1.0
        p.do_sample, p.temperature, p.top_k = int(gen.do_sample), float(gen.temperature), int(gen.top_k)
        p.top_p, p.epsilon_cutoff, p.seed = float(gen.top_p), float(gen.epsilon_cutoff), int(gen.seed)
        sid_arr = (C.c_int * n)(*stream_ids)
        # every int32 sequence of the call lives in ONE buffer per argument, the per-stream pointers are offsets into it (64 streams: the
        # marshalling is host time during which the GPU idles between two steps)
        keep_p, prompt_ptrs, prompt_lens = _pack_int32(prompt_ids, n)
        keep_v, prev_ptrs, prev_lens = _pack_int32(prev_target_ids, n)
        keep_f, forced_ptrs, forced_lens = _pack_int32([None] * n if forced_tokens is None else forced_tokens, n)
        outs = np.zeros((n, max(1, gen.max_new_tokens)), dtype=np.int32)
        out_base, out_stride = outs.ctypes.data, outs.strides[0]
        out_ptrs = (C.c_void_p * n)(*[out_base + i * out_stride for i in range(n)])
        out_lens = (C.c_int * n)()
        logits = np.zeros((n, gen.max_new_tokens, self.cfg.vocab), dtype=np.float32) if return_logits else None
        if on_device:
            pcm_ptrs = (C.c_void_p * n)(*[x.data_ptr() for x in pcm])
        else:
            pcm_ptrs = (C.c_void_p * n)(*[x.ctypes.data for x in pcm])
        args = (self.h, C.byref(p), n, sid_arr, pcm_ptrs, n_samples, prompt_ptrs, prompt_lens, prev_ptrs, prev_lens, forced_ptrs, forced_lens,
                out_ptrs, out_lens, None if logits is None else logits.ctypes.data, _stream_ptr())
        t0 = time.perf_counter()
        rc = self.lib.isst_generate(*args)
        self.last_call_seconds = time.perf_counter() - t0  # wall time inside the library (it returns once the last token id is on the host)
        self._check(rc, "isst_generate")
        del keep_p, keep_v, keep_f
        rows = outs.tolist()
        return [rows[i][: out_lens[i]] for i in range(n)], logits

    def encode_speech(self, sid: int, pcm: np.ndarray, multiplier: int = 1) -> torch.Tensor:
        """speech_encoder.encode_speech for one stream -> (S, llm_dim) bf16 CPU tensor (test aid)."""
        pcm = np.ascontiguousarray(pcm, dtype=np.float32)
        S_max = pcm.shape[0] // (self.cfg.samples_per_frame * self.cfg.shrink_factor)
        out = torch.empty((S_max, self.cfg.llm_dim), dtype=torch.bfloat16)
        rows = C.c_int(0)
        self._check(self.lib.isst_encode_speech(self.h, sid, pcm.ctypes.data, pcm.shape[0], multiplier, out.data_ptr(),
                                                C.byref(rows), _stream_ptr()), "isst_encode_speech")
        return out[: rows.value]

    def read_kv(self, sid: int, pos: int, layer: int = 0, kv_head: int = 0, beam: int = 0):
        """(K, V) rows (128 bf16 each, unrotated) of one cached position (test aid)."""
        k = torch.empty(128, dtype=torch.bfloat16)
        v = torch.empty(128, dtype=torch.bfloat16)
        self._check(self.lib.isst_debug_read_kv(self.h, sid, beam, layer, kv_head, pos, k.data_ptr(), v.data_ptr()), "isst_debug_read_kv")
        return k, v

    def profile_begin(self, rows_lo: int = 1, rows_hi: int = 1):
        """Bracket the gate/up launch of every Llama pass of rows_lo..rows_hi rows (default: the one-token decode GEMV)."""
        self._check(self.lib.isst_profile_begin_rows(self.h, rows_lo, rows_hi), "isst_profile_begin_rows")

    def profile_end(self):
        """(average event bracket in us around the profiled gate/up launches, launches timed) since profile_begin."""
        avg, n = C.c_double(0.0), C.c_int64(0)
        self._check(self.lib.isst_profile_end(self.h, _stream_ptr(), C.byref(avg), C.byref(n)), "isst_profile_end")
        return avg.value, n.value

    def debug_tap(self, name: str) -> torch.Tensor:
        got = C.c_int64(0)
        self._check(self.lib.isst_debug_tap(self.h, name.encode(), None, 0, C.byref(got)), f"isst_debug_tap({name})")
        out = torch.empty(got.value, dtype=torch.bfloat16)
        self._check(self.lib.isst_debug_tap(self.h, name.encode(), out.data_ptr(), got.value, C.byref(got)),
                    "isst_debug_tap")
        return out


# -------------------------------------------------------------------- per-kernel wrappers (device tensors)
def op_pack_weight(w: torch.Tensor, conv_k: int = 0) -> torch.Tensor:
    lib = load_library()
    n_rows = w.shape[0]
    K = w.numel() // n_rows
    out = torch.zeros(lib.isst_op_packed_elems(n_rows, K), dtype=torch.bfloat16, device=w.device)
    rc = lib.isst_op_pack_weight(_ptr(w.contiguous()), _ptr(out), n_rows, K, conv_k, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_pack_weight -> {rc}")
    return out


def op_pack_gateup8(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """gate_proj / up_proj (ffn, K) as self-paired tiles for op_gemm(..., N=2 * ffn, epi="swiglu8")."""
    lib = load_library()
    ffn, K = gate.shape
    out = torch.zeros(2 * ffn * K, dtype=torch.bfloat16, device=gate.device)
    rc = lib.isst_op_pack_gateup8(_ptr(gate.contiguous()), _ptr(up.contiguous()), _ptr(out), ffn, K, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_pack_gateup8 -> {rc}")
    return out


def op_gemm(A: torch.Tensor, packed: torch.Tensor, N: int, epi: str = "none", bias=None, res=None, n_valid=None,
            lda: Optional[int] = None, M: Optional[int] = None, K: Optional[int] = None, norm_w=None,
            norm_eps: float = 1e-5) -> torch.Tensor:
    lib = load_library()
    M = A.shape[0] if M is None else M
    K = A.shape[1] if K is None else K
    lda = A.stride(0) if lda is None else lda
    n_out = (N // 2 if epi in ("swiglu", "swiglu8") else N) if n_valid is None else n_valid
    out = torch.zeros((M, n_out), dtype=torch.float32 if epi == "f32" else torch.bfloat16, device=A.device)
    rc = lib.isst_op_gemm(_ptr(A), lda, _ptr(packed), _ptr(bias), _ptr(res), 0 if res is None else res.stride(0),
                          _ptr(out), out.stride(0), M, N, K, n_out, EPI[epi], _ptr(norm_w), norm_eps, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_gemm -> {rc}")
    return out


def dense_kernel_name() -> str:
    """The kernel isst_op_gemm dispatches to above 64 rows (bench.py's `mfma` block names it)."""
    return "gemm_dense_kernel<EPI> (256 x 256 tile, 8-wave ping-pong, LDS-DMA; gemm_dense.hip)"


def op_gemm_splitk_rmsnorm(A: torch.Tensor, packed: torch.Tensor, x: torch.Tensor, ksplit: int, norm_w=None, norm_eps: float = 1e-5):
    """x <- bf16(x + bf16(A @ W^T)) through `ksplit` fp32 K-slabs; returns (x_new, RMSNorm(x_new) or None).  17..64 rows."""
    lib = load_library()
    M, K = A.shape
    N = x.shape[1]
    x = x.clone()
    out = torch.empty_like(x) if norm_w is not None else None
    slabs = torch.empty((ksplit, M, N), dtype=torch.float32, device=A.device)
    rc = lib.isst_op_gemm_splitk_rmsnorm(_ptr(A), A.stride(0), _ptr(packed), _ptr(x), _ptr(norm_w), _ptr(out), _ptr(slabs), M, N, K,
                                         ksplit, norm_eps, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_gemm_splitk_rmsnorm -> {rc}")
    return x, out


def op_gemm_splitk_fused(A: torch.Tensor, packed: torch.Tensor, x: torch.Tensor, ksplit: int, tickets: Optional[torch.Tensor] = None):
    """The launch-free form of op_gemm_splitk_rmsnorm's first half: returns (x_new, ssq [M][N/32] fp32, tickets) -- 13..64 rows."""
    lib = load_library()
    M, K = A.shape
    N = x.shape[1]
    x = x.clone()
    slabs = torch.empty((ksplit, M, N), dtype=torch.float32, device=A.device)
    ssq = torch.zeros((M, N // 32), dtype=torch.float32, device=A.device)
    if tickets is None:
        tickets = torch.zeros(N // 16, dtype=torch.int32, device=A.device)
    lib.isst_op_gemm_splitk_fused.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p]
    rc = lib.isst_op_gemm_splitk_fused(_ptr(A), A.stride(0), _ptr(packed), _ptr(x), _ptr(slabs), _ptr(ssq), _ptr(tickets), M, N, K, ksplit, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_gemm_splitk_fused -> {rc}")
    return x, ssq, tickets


def op_gemm_splitk_plain(A: torch.Tensor, packed: torch.Tensor, N: int, ksplit: int, norm_w=None, ssq=None, norm_eps: float = 1e-5):
    """bf16(A @ W^T) through `ksplit` K slices reduced inside the launch (no residual); norm_w + ssq: A rows RMS-normalised while staged."""
    lib = load_library()
    M, K = A.shape
    out = torch.zeros((M, N), dtype=torch.bfloat16, device=A.device)
    slabs = torch.empty((ksplit, M, N), dtype=torch.float32, device=A.device)
    tickets = torch.zeros(N // 16, dtype=torch.int32, device=A.device)
    lib.isst_op_gemm_splitk_plain.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int,
                                              C.c_void_p, C.c_float, C.c_void_p, C.c_void_p]
    rc = lib.isst_op_gemm_splitk_plain(_ptr(A), A.stride(0), _ptr(packed), _ptr(out), out.stride(0), _ptr(slabs), _ptr(tickets), M, N, K, ksplit,
                                       _ptr(norm_w), norm_eps, _ptr(ssq), _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_gemm_splitk_plain -> {rc}")
    assert int(tickets.abs().sum()) == 0, "arrival counters not re-armed"
    return out


def op_gemm_norm_ssq(x: torch.Tensor, packed: torch.Tensor, N: int, norm_w: torch.Tensor, ssq: torch.Tensor, epi: str = "none", norm_eps: float = 1e-5):
    """epi(RMSNorm(x) @ W^T) with the rows normalised while they are staged (1/rms from the producer's sums of squares) -- 13..64 rows."""
    lib = load_library()
    M, K = x.shape
    n_out = N // 2 if epi == "swiglu" else N
    out = torch.zeros((M, n_out), dtype=torch.float32 if epi == "f32" else torch.bfloat16, device=x.device)
    lib.isst_op_gemm_norm_ssq.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_float, C.c_void_p, C.c_void_p]
    rc = lib.isst_op_gemm_norm_ssq(_ptr(x), x.stride(0), _ptr(packed), _ptr(out), out.stride(0), M, N, K, n_out, EPI[epi], _ptr(norm_w), norm_eps, _ptr(ssq), _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_gemm_norm_ssq -> {rc}")
    return out


def op_gemm_splitk_layernorm(A, packed, bias, x, ksplit, ln_w, ln_b, eps=1e-5):
    """x <- bf16(x + bf16(A @ W^T + bias)) through `ksplit` fp32 K-slabs; returns (x_new, LayerNorm(x_new))."""
    lib = load_library()
    M, K = A.shape
    N = x.shape[1]
    x = x.clone()
    out = torch.empty_like(x)
    slabs = torch.empty((ksplit, M, N), dtype=torch.float32, device=A.device)
    rc = lib.isst_op_gemm_splitk_layernorm(_ptr(A), A.stride(0), _ptr(packed), _ptr(bias), _ptr(x), _ptr(ln_w), _ptr(ln_b), _ptr(out), _ptr(slabs),
                                           M, N, K, ksplit, eps, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_gemm_splitk_layernorm -> {rc}")
    return x, out


def op_layernorm(x, w, b, eps=1e-5, gelu=False):
    lib = load_library()
    out = torch.empty_like(x)
    rc = lib.isst_op_layernorm(_ptr(x), _ptr(w), _ptr(b), _ptr(out), x.shape[0], x.shape[1], eps, int(gelu), _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_layernorm -> {rc}")
    return out


def op_rmsnorm(x, w, eps=1e-5):
    lib = load_library()
    out = torch.empty_like(x)
    rc = lib.isst_op_rmsnorm(_ptr(x), _ptr(w), _ptr(out), x.shape[0], x.shape[1], eps, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_rmsnorm -> {rc}")
    return out


def op_conv0(audio, w, bias, ln_w, ln_b, k, stride):
    lib = load_library()
    Cc = w.shape[0]
    T = (audio.shape[0] - k) // stride + 1
    out = torch.empty((T, Cc), dtype=torch.bfloat16, device=audio.device)
    rc = lib.isst_op_conv0(_ptr(audio), _ptr(w.contiguous()), _ptr(bias), _ptr(ln_w), _ptr(ln_b), _ptr(out), T, Cc, k,
                           stride, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_conv0 -> {rc}")
    return out


def op_sample(logits: torch.Tensor, ids, enc_ids, suppress, penalty, ngram, enc_ngram) -> int:
    lib = load_library()
    dev = logits.device

    def mk(x):
        return torch.tensor(list(x) if len(x) else [0], dtype=torch.int32, device=dev)

    ids_t, enc_t, sup_t = mk(ids), mk(enc_ids), mk(suppress)
    out = torch.zeros(1, dtype=torch.int32, device=dev)
    rc = lib.isst_op_sample(_ptr(logits), logits.numel(), _ptr(ids_t), len(ids), _ptr(enc_t), len(enc_ids), _ptr(sup_t),
                            len(suppress), penalty, ngram, enc_ngram, _ptr(out), _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_sample -> {rc}")
    return int(out.item())


def op_warp_sample(scores: np.ndarray, temperature: float, top_k: int, top_p: float, epsilon_cutoff: float, u: float):
    """HF's warpers Temperature -> TopK -> TopP -> Epsilon on one row of processed scores + the inverse-CDF draw (host code: no GPU needed).
    Returns (warped scores, token)."""
    lib = load_library()
    s = np.ascontiguousarray(scores, dtype=np.float32).copy()
    tok = C.c_int(-1)
    rc = lib.isst_op_warp_sample(s.ctypes.data, s.size, temperature, top_k, top_p, epsilon_cutoff, u, C.byref(tok))
    if rc:
        raise IsstError(f"isst_op_warp_sample -> {rc}")
    return s, tok.value


def op_warp(scores: np.ndarray, temperature: float, top_k: int, top_p: float, epsilon_cutoff: float, min_tokens_to_keep: int = 1) -> np.ndarray:
    """HF's warpers on one row of processed scores (host code: csrc/warp.hip); returns the warped copy."""
    lib = load_library()
    s = np.ascontiguousarray(scores, dtype=np.float32).copy()
    lib.isst_op_warp.argtypes = [C.c_void_p, C.c_int, C.c_float, C.c_int, C.c_float, C.c_float, C.c_int]
    rc = lib.isst_op_warp(s.ctypes.data, s.size, temperature, top_k, top_p, epsilon_cutoff, min_tokens_to_keep)
    if rc:
        raise IsstError(f"isst_op_warp -> {rc}")
    return s


def op_multinomial_wor(scores: np.ndarray, k: int, uniforms: Sequence[float]) -> list:
    """`torch.multinomial(softmax(scores), k)` without replacement as k sequential inverse-CDF draws at the given uniforms (host code: csrc/warp.hip)."""
    lib = load_library()
    s = np.ascontiguousarray(scores, dtype=np.float32)
    u = np.ascontiguousarray(uniforms, dtype=np.float64)
    out = np.zeros(k, dtype=np.int64)
    lib.isst_op_multinomial_wor.argtypes = [C.c_void_p, C.c_long, C.c_int, C.c_void_p, C.c_void_p]
    rc = lib.isst_op_multinomial_wor(s.ctypes.data, s.size, k, u.ctypes.data, out.ctypes.data)
    if rc:
        raise IsstError(f"isst_op_multinomial_wor -> {rc}")
    return out.tolist()


def op_sample_uniform(seed: int, stream: int, chunk: int, step: int) -> float:
    return float(load_library().isst_op_sample_uniform(seed, stream, chunk, step))


def op_splice_map(ids: Sequence[int], user_id: int, assistant_id: int, start_header_id: int, n_features: int) -> list:
    """Row map of the speech splice (host logic of the library): entry >= 0 = prompt token index, < 0 = speech feature -1 - entry."""
    lib = load_library()
    a = np.ascontiguousarray(np.asarray(ids, dtype=np.int32))
    out = np.zeros(a.size, dtype=np.int32)
    n = C.c_int(0)
    rc = lib.isst_op_splice_map(a.ctypes.data, a.size, user_id, assistant_id, start_header_id, n_features, out.ctypes.data, C.byref(n))
    if rc:
        raise IsstError(f"isst_op_splice_map -> {rc}")
    return out[: n.value].tolist()


def op_embed_splice(ids: torch.Tensor, speech_row: Optional[torch.Tensor], table: torch.Tensor, speech: Optional[torch.Tensor]) -> torch.Tensor:
    """out[r] = speech[speech_row[r]] if speech_row[r] >= 0 else table[ids[r]] (int32 device tensors, bf16 tables)."""
    lib = load_library()
    rows, D = ids.numel(), table.shape[1]
    out = torch.empty((rows, D), dtype=torch.bfloat16, device=table.device)
    rc = lib.isst_op_embed_splice(_ptr(ids), _ptr(speech_row), _ptr(table), _ptr(speech), _ptr(out), rows, D, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_embed_splice -> {rc}")
    return out


def op_enc_attention(qkv: torch.Tensor, kring: torch.Tensor, vring: torch.Tensor, ring_start: int, prefix: int, rope_cos: torch.Tensor,
                     rope_sin: torch.Tensor, round_each: bool, heads: int, max_cache: int, blocksize: int) -> torch.Tensor:
    """qkv (Q, 3*heads*64) bf16; kring (heads, cap, 64), vring (heads, 64, cap) are updated in place; -> (Q, heads*64)."""
    lib = load_library()
    Q, cap = qkv.shape[0], kring.shape[1]
    out = torch.empty((Q, heads * 64), dtype=torch.bfloat16, device=qkv.device)
    rc = lib.isst_op_enc_attention(_ptr(qkv), _ptr(kring), _ptr(vring), ring_start, prefix, _ptr(rope_cos), _ptr(rope_sin), int(round_each), _ptr(out),
                                   Q, heads, cap, max_cache, blocksize, _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_enc_attention -> {rc}")
    return out


def op_llm_attention(qkv: torch.Tensor, pos0: int, kpool: torch.Tensor, krpool: torch.Tensor, vpool: torch.Tensor, heads: int, kv_heads: int,
                     sys_cap: int, ring_cap: int, sys_len: int, ring_start: int, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
                     rot_keys: bool = True) -> torch.Tensor:
    """qkv (rows, (heads + 2 kv_heads) * 128) bf16 at positions pos0..; pools (kv_heads, sys_cap + ring_cap, 128) updated in place;
    rope tables bf16 (>= pos0 + rows, 64); -> (rows, heads * 128)."""
    lib = load_library()
    rows = qkv.shape[0]
    out = torch.empty((rows, heads * 128), dtype=torch.bfloat16, device=qkv.device)
    rc = lib.isst_op_llm_attention(_ptr(qkv), rows, pos0, _ptr(kpool), _ptr(krpool), _ptr(vpool), heads, kv_heads, sys_cap, ring_cap, sys_len, ring_start,
                                   _ptr(rope_cos), _ptr(rope_sin), int(rot_keys), _ptr(out), _stream_ptr())
    if rc:
        raise IsstError(f"isst_op_llm_attention -> {rc}")
    return out


# ---------------------------------------------------------------- a decode step of many streams over one prompt
# (these functions cost a decode step some ten microseconds of host time each next to kernels that take as long: their checks are written for the call that passes)
def _device_of(what: str, t: torch.Tensor) -> int:
    if t.get_device() < 0 or not t.is_cuda:
        raise IsstError(f"{what}: tensors must be on a GPU, got {t.device}")
    return t.get_device()


def _expect(what: str, dev: int, name: str, t: torch.Tensor, dtype: torch.dtype, shape, contiguous: bool = True):
    if t.dtype is not dtype or t.shape != shape:
        raise IsstError(f"{what}: {name} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != dev:
        raise IsstError(f"{what}: {name} is on {t.device}, expected cuda:{dev}")
    if contiguous and not t.is_contiguous():
        raise IsstError(f"{what}: {name} must be contiguous (strides {t.stride()})")


def _row_strides(what: str, name: str, t: torch.Tensor):
    """Strides of all dims but the last (0 where a dim has no second entry), for rows the kernels read 16 bytes at a time."""
    if t.numel() == 0:
        return (0,) * (t.dim() - 1)
    st = tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]))
    if (t.stride(-1) != 1 and t.shape[-1] > 1) or t.data_ptr() % 16 or any(s % 8 for s in st):
        raise IsstError(f"{what}: rows of {name} must be contiguous and 16-byte aligned (strides {t.stride()})")
    return st


def _launch(what: str, dev: int, workspace_bytes: int, call):
    """call(workspace pointer, bytes, stream) on the current stream of `dev`; the workspace is the caching allocator's, i.e. ordered by that stream."""
    if workspace_bytes < 0:
        raise IsstError(f"{what}: bad arguments ({workspace_bytes})")
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _launch(what, dev, workspace_bytes, call)
    ws = torch.empty(workspace_bytes, dtype=torch.uint8, device=dev) if workspace_bytes else None
    rc = call(None if ws is None else ws.data_ptr(), workspace_bytes, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        raise IsstError(f"{what} -> {rc}")


def op_prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k_tail: torch.Tensor, v_tail: torch.Tensor, tail_lens: torch.Tensor,
                        row_starts: Optional[torch.Tensor] = None, max_rows: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of sequences that share the keys k_prefix / v_prefix (kv_heads, P, D) in front of their own k_tail / v_tail (seqs, kv_heads, cap, D), of which
    tail_lens (seqs, int32) are live.  q (rows, heads, D): sequence b's newest positions are rows row_starts[b] .. row_starts[b + 1] - 1 (int32, seqs + 1; None: as many
    rows each); row t of n sees the prefix and the own keys 0 .. tail_lens[b] - n + t, a row without a key gives zeros, a row of no sequence is left as it was (in `out`;
    undefined without).  max_rows: most rows of one sequence if the caller knows it (speed only).  bf16, D 64 or 128, keys already rotated; strided views are fine while
    rows are 16-byte aligned (out: [rows][heads] or [heads][rows]).  Softmax weights enter the value product as bf16, all else is fp32.  scale: default D ** -0.5."""
    what = "op_prefix_attention"
    lib = _lib or load_library()
    dev = _device_of(what, q)
    if q.dim() != 3 or k_prefix.dim() != 3 or k_tail.dim() != 4:
        raise IsstError(f"{what}: q (rows, heads, D), k_prefix (kv_heads, P, D), k_tail (seqs, kv_heads, cap, D), got {tuple(q.shape)}, {tuple(k_prefix.shape)}, {tuple(k_tail.shape)}")
    bf = torch.bfloat16
    (rows, heads, D), (kv, P, _), (seqs, _, cap, _) = q.shape, k_prefix.shape, k_tail.shape
    prefix, tail = (kv, P, D), (seqs, kv, cap, D)
    if not (q.dtype is bf and k_prefix.dtype is bf and v_prefix.dtype is bf and k_tail.dtype is bf and v_tail.dtype is bf and tail_lens.dtype is torch.int32
            and v_prefix.shape == prefix and k_prefix.shape == prefix and k_tail.shape == tail and v_tail.shape == tail and tail_lens.shape == (seqs,)
            and k_prefix.get_device() == dev and v_prefix.get_device() == dev and k_tail.get_device() == dev and v_tail.get_device() == dev
            and tail_lens.get_device() == dev and tail_lens.is_contiguous()):
        for name, t, shape in (("q", q, q.shape), ("k_prefix", k_prefix, prefix), ("v_prefix", v_prefix, prefix), ("k_tail", k_tail, tail), ("v_tail", v_tail, tail)):
            _expect(what, dev, name, t, bf, shape, False)
        _expect(what, dev, "tail_lens", tail_lens, torch.int32, (seqs,))
    if row_starts is not None:
        _expect(what, dev, "row_starts", row_starts, torch.int32, (seqs + 1,))
    if out is None:
        out = q.new_empty((rows, heads, D))
    else:
        _expect(what, dev, "out", out, bf, (rows, heads, D), False)
    if D not in (64, 128) or kv < 1 or heads < 1 or heads % kv or (rows and not seqs) or (row_starts is None and seqs and rows % seqs) or max_rows < 0:
        raise IsstError(f"{what}: {rows} rows of {seqs} sequences, {heads} heads on {kv} key heads of {D} (max_rows {max_rows}) are not supported")
    pq, po, pkp, pvp, pkt, pvt = q.data_ptr(), out.data_ptr(), k_prefix.data_ptr(), v_prefix.data_ptr(), k_tail.data_ptr(), v_tail.data_ptr()
    (q0, q1, q2), (o0, o1, o2), (kp0, kp1, kp2), (vp0, vp1, vp2) = q.stride(), out.stride(), k_prefix.stride(), v_prefix.stride()
    (kt0, kt1, kt2, kt3), (vt0, vt1, vt2, vt3) = k_tail.stride(), v_tail.stride()
    if (q2 != 1 or o2 != 1 or kp2 != 1 or vp2 != 1 or kt3 != 1 or vt3 != 1 or (q0 | q1 | o0 | o1 | kp0 | kp1 | vp0 | vp1 | kt0 | kt1 | kt2 | vt0 | vt1 | vt2) & 7
            or (pq | po | pkp | pvp | pkt | pvt) & 15):  # (mostly dims of one entry or none, whose strides do not count)
        (q0, q1), (o0, o1), (kp0, kp1), (vp0, vp1), (kt0, kt1, kt2), (vt0, vt1, vt2) = (
            _row_strides(what, n, t) for n, t in (("q", q), ("out", out), ("k_prefix", k_prefix), ("v_prefix", v_prefix), ("k_tail", k_tail), ("v_tail", v_tail)))
    a = _PrefixAttn(pq, pkp, pvp, pkt, pvt, tail_lens.data_ptr(), None if row_starts is None else row_starts.data_ptr(), po, q0, q1, o0, o1, kp0, kp1, vp0, vp1, kt0, kt1, kt2,
                    vt0, vt1, vt2, rows, seqs, max_rows, heads, kv, D, P, cap, D ** -0.5 if scale is None else scale)
    ref = C.byref(a)
    _launch(what, dev, lib.isst_op_prefix_attention_workspace(ref), lambda ws, n, st: lib.isst_op_prefix_attention(ref, ws, n, st))
    return out


def op_gemm_lora(x: torch.Tensor, packed: torch.Tensor, N: int, down: torch.Tensor, up: torch.Tensor, scales: torch.Tensor, row_adapter: torch.Tensor,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """bf16(x W^T + scales[a] (x down[a]^T) up[a]^T) with a = row_adapter[m] per row (int32; outside 0 .. n - 1: no adapter).  x (M, K) bf16, packed = op_pack_weight(W (N, K)),
    down (n, rank, K), up (n, N, rank) bf16, scales (n,) fp32; rank a multiple of 8 up to 128 (pad smaller ones with zeros), K a multiple of 32."""
    what = "op_gemm_lora"
    lib = _lib or load_library()
    dev = _device_of(what, x)
    if x.dim() != 2 or down.dim() != 3:
        raise IsstError(f"{what}: x (M, K), down (n, rank, K), got {tuple(x.shape)}, {tuple(down.shape)}")
    bf = torch.bfloat16
    (M, K), (n, rank, _) = x.shape, down.shape
    image = (N + 15) // 16 * 16 * K
    if not (x.dtype is bf and packed.dtype is bf and down.dtype is bf and up.dtype is bf and scales.dtype is torch.float32 and row_adapter.dtype is torch.int32
            and packed.shape == (image,) and up.shape == (n, N, rank) and scales.shape == (n,) and row_adapter.shape == (M,)
            and packed.get_device() == dev and down.get_device() == dev and up.get_device() == dev and scales.get_device() == dev and row_adapter.get_device() == dev
            and packed.is_contiguous() and down.is_contiguous() and up.is_contiguous() and scales.is_contiguous() and row_adapter.is_contiguous()):
        _expect(what, dev, "x", x, bf, (M, K), False)
        _expect(what, dev, "packed", packed, bf, (image,))
        _expect(what, dev, "down", down, bf, (n, rank, K))
        _expect(what, dev, "up", up, bf, (n, N, rank))
        _expect(what, dev, "scales", scales, torch.float32, (n,))
        _expect(what, dev, "row_adapter", row_adapter, torch.int32, (M,))
    if out is None:
        out = x.new_empty((M, N))
    else:
        _expect(what, dev, "out", out, bf, (M, N), False)
        if (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise IsstError(f"{what}: rows of out must be contiguous and apart (strides {out.stride()})")
    lda = x.stride(0)
    if x.stride(1) != 1 or lda & 7:
        (lda,) = _row_strides(what, "x", x)
    if M > 1 and lda < K:
        raise IsstError(f"{what}: rows of x overlap (strides {x.stride()})")
    _launch(what, dev, lib.isst_op_gemm_lora_workspace(M, N, K, rank, n),
            lambda ws, nb, st: lib.isst_op_gemm_lora(x.data_ptr(), lda if M > 1 else K, packed.data_ptr(), down.data_ptr(), up.data_ptr(), scales.data_ptr(),
                                                     row_adapter.data_ptr(), n, rank, out.data_ptr(), out.stride(0) if M > 1 else N, M, N, K, ws, nb, st))
    return out


def op_verify_drafts(target: torch.Tensor, drafts: torch.Tensor, n_drafts: Optional[torch.Tensor] = None, draft_scores: Optional[torch.Tensor] = None,
                     uniforms: Optional[torch.Tensor] = None):
    """Drafted tokens against the model's scores: target (streams, K + 1, vocab) fp32 processed scores (-inf = removed), drafts (streams, K) int32 of which n_drafts[b] (None: all)
    are live, draft_scores (streams, K, vocab) fp32 or None (a draft without a distribution), uniforms (streams, K + 1) float64 in [0, 1) -- [:, i] decides draft i, [:, K] draws the
    token behind the last accepted one -- or None: greedy.  Returns (tokens (streams, K + 1) int32: accepted drafts, next token, -1 behind them; counts (streams,) int32, -1 for a
    stream whose deciding row has no distribution or whose inputs are out of range)."""
    what = "op_verify_drafts"
    lib = _lib or load_library()
    dev = _device_of(what, target)
    if target.dim() != 3 or target.shape[1] < 1 or target.shape[2] < 1:
        raise IsstError(f"{what}: target (streams, K + 1, vocab), got {tuple(target.shape)}")
    B, K, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    _expect(what, dev, "target", target, torch.float32, (B, K + 1, V), False)
    _expect(what, dev, "drafts", drafts, torch.int32, (B, K))
    if n_drafts is not None:
        _expect(what, dev, "n_drafts", n_drafts, torch.int32, (B,))
    if draft_scores is not None:
        _expect(what, dev, "draft_scores", draft_scores, torch.float32, (B, K, V), False)
    if uniforms is not None:
        _expect(what, dev, "uniforms", uniforms, torch.float64, (B, K + 1))
    if uniforms is None and draft_scores is not None:
        raise IsstError(f"{what}: greedy verification reads no draft scores")
    t_st, d_st = target.stride(), (0, 0, 1) if draft_scores is None else draft_scores.stride()
    if V > 1 and (t_st[2] != 1 or d_st[2] != 1):
        raise IsstError(f"{what}: rows of the scores must be contiguous (strides {t_st}, {d_st})")
    tokens, counts = drafts.new_empty((B, K + 1)), drafts.new_empty((B,))
    ptr = lambda t: None if t is None else t.data_ptr()
    _launch(what, dev, lib.isst_op_verify_drafts_workspace(B, K, V),
            lambda ws, n, st: lib.isst_op_verify_drafts(target.data_ptr(), t_st[0], t_st[1], ptr(draft_scores), d_st[0], d_st[1], drafts.data_ptr(), ptr(n_drafts), ptr(uniforms),
                                                        B, K, V, tokens.data_ptr(), counts.data_ptr(), ws, n, st))
    return tokens, counts
