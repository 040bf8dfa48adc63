"""Kernel entry points.  ``from pulse_infer_b200 import ops`` then ``ops.embed(...)`` and so on."""
from . import kernels
from .kernels import (BF16, F32, SPLIT_KEYS, DECODE_MAX_SEGMENTS, KernelError, NormedRows, add_rmsnorm, argmax, attention_mma, attention_num_splits, attention_splits_bound, choose_prompt_splits, choose_split_keys,
                      attention_simple, attention_decode_fused, attention_decode_fused_usable, attention_decode_workspace, decode_on_tcgen05, DecodeWorkspace, attention_tcgen05, attention_tcgen05_status, attention_tcgen05_loaded_status, attention_tcgen05_usable, attention_decode_tcgen05_usable, embed, gemm_f32, gemm_small_m, gemm_tcgen05, gemm_tcgen05_status, interleave_gate_up, linear, logit_edit, logit_rules, preload, qk_norm_rope_write, rope_table,
                      sample, sample_entries, silu_mul, small_m_usable)
from .cache_8bit import (BLOCK_TOKENS, CACHE_8BIT_DTYPES, DECODE_8BIT_MAX_SEGMENTS, PAGE_MAPS_MAX_SEGMENTS, PageMaps, attention_decode_8bit, attention_prompt_8bit, cache_8bit_pools,
                         cache_8bit_usable, page_maps, pages_8bit_to_bf16, qk_norm_rope_write_8bit)

__all__ = ["BLOCK_TOKENS", "CACHE_8BIT_DTYPES", "DECODE_8BIT_MAX_SEGMENTS", "PAGE_MAPS_MAX_SEGMENTS", "PageMaps", "attention_decode_8bit", "attention_prompt_8bit", "cache_8bit_pools",
           "cache_8bit_usable", "page_maps", "pages_8bit_to_bf16", "qk_norm_rope_write_8bit", "logit_rules",
           "DECODE_MAX_SEGMENTS", "BF16", "F32", "SPLIT_KEYS", "KernelError", "NormedRows", "add_rmsnorm", "argmax", "attention_mma",
           "attention_num_splits", "attention_splits_bound", "choose_prompt_splits", "choose_split_keys", "attention_simple", "attention_decode_fused", "attention_decode_fused_usable", "attention_decode_workspace", "decode_on_tcgen05", "DecodeWorkspace", "attention_tcgen05", "attention_tcgen05_status", "attention_tcgen05_loaded_status", "attention_tcgen05_usable", "attention_decode_tcgen05_usable", "embed", "gemm_f32", "gemm_small_m", "gemm_tcgen05", "gemm_tcgen05_status", "interleave_gate_up", "linear", "logit_edit", "preload",
           "qk_norm_rope_write", "rope_table", "sample", "sample_entries", "silu_mul", "small_m_usable"]
