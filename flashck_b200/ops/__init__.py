"""Functional operations (the reference's ``flash_ck.ops``), attention family only."""
from . import fmha
from .fmha import (batch_prefill, default_num_splits, fmha_fwd, fmha_fwd_append_kv, fmha_fwd_fp8,
                   fmha_fwd_paged_kv_prefill, fmha_fwd_splitkv, fmha_fwd_splitkv_combine,
                   fmha_fwd_splitkv_combine_strided, fmha_fwd_var_len, quantize_fp8, splitkv_workspace)
from .gradients import fmha_autograd, fmha_autograd_var_len, fmha_bwd, fmha_bwd_var_len
from .int4 import fmha_fwd_append_kv_int4, fmha_fwd_splitkv_int4, fmha_read_kv_int4, int4_cache
from .rotary import apply_rotary, apply_rotary_autograd
from .shared_prefix import fmha_fwd_shared_prefix

__all__ = [
    "fmha", "fmha_fwd", "fmha_fwd_var_len", "fmha_fwd_fp8", "quantize_fp8", "batch_prefill", "fmha_fwd_paged_kv_prefill", "fmha_fwd_splitkv",
    "fmha_fwd_splitkv_combine", "fmha_fwd_splitkv_combine_strided", "fmha_fwd_append_kv", "splitkv_workspace", "default_num_splits",
    "fmha_bwd", "fmha_bwd_var_len", "fmha_autograd", "fmha_autograd_var_len", "fmha_fwd_shared_prefix",
    "int4_cache", "fmha_fwd_append_kv_int4", "fmha_fwd_splitkv_int4", "fmha_read_kv_int4", "apply_rotary", "apply_rotary_autograd",
]
