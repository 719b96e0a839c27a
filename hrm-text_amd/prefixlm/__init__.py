"""MI355X-native packed varlen PrefixLM attention (HRM-Text hot path).

Public names follow the reference module models/flash_attention_prefixlm_v2.py.
"""
from .metadata import compute_aux_seq_tensors_scalars, useful_entries, useful_flops
from .op import FlashAttnVarlenPrefixLM, flash_attn_varlen_prefixlm
from .plan import build_plan, plan_ds_blocks, plan_inputs, plan_size
from .layer import fused_attention_layer
from .kvcache import flash_attn_with_kvcache
from .kvcache8 import KVCacheQ8, flash_attn_with_kvcache_q8, kvcache_q8
from .norm_mlp import rms_norm, swiglu
from .embedding import embedding
from .logprob import TokenLogprobs, token_logprobs

__all__ = [
    "build_plan",
    "compute_aux_seq_tensors_scalars",
    "embedding",
    "flash_attn_varlen_prefixlm",
    "flash_attn_with_kvcache",
    "flash_attn_with_kvcache_q8",
    "fused_attention_layer",
    "FlashAttnVarlenPrefixLM",
    "KVCacheQ8",
    "kvcache_q8",
    "TokenLogprobs",
    "token_logprobs",
    "useful_entries",
    "useful_flops",
    "plan_ds_blocks",
    "plan_inputs",
    "plan_size",
    "rms_norm",
    "swiglu",
]
