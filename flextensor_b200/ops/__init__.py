"""Hand-written sm_100a kernels (tcgen05 GEMM, flash attention, norms/RoPE, fused
tensor/context-parallel collectives) and their Python entry points."""

from flextensor_b200.ops.api import (
    EPI,
    TP_EPI,
    attention,
    attention_cp,
    decode_attention,
    decode_attention_q8,
    kv_append_q8,
    launch_count,
    layernorm_modulate,
    linear,
    linear_swiglu,
    MOE_DECODE_MAX_EXPERTS,
    MOE_DECODE_MAX_TOKENS,
    MOE_DECODE_MAX_TOPK,
    moe_decode,
    qk_rmsnorm_rope,
    rmsnorm,
    rope,
    tp_ag_counter_words,
    tp_allgather_gemm,
    tp_gemm_reducescatter,
    tp_reduce,
    tp_rmsnorm,
)

__all__ = ["EPI", "TP_EPI", "attention", "attention_cp", "decode_attention", "decode_attention_q8", "kv_append_q8", "launch_count", "layernorm_modulate", "linear",
           "linear_swiglu", "MOE_DECODE_MAX_EXPERTS", "MOE_DECODE_MAX_TOKENS", "MOE_DECODE_MAX_TOPK", "moe_decode", "qk_rmsnorm_rope", "rmsnorm", "rope", "tp_ag_counter_words", "tp_allgather_gemm", "tp_gemm_reducescatter",
           "tp_reduce", "tp_rmsnorm"]
