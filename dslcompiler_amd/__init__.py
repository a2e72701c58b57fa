"""MI355X (gfx950) backend for DSLCompiler's fused SwiGLU / micro.mma path.

The product is ``libllk_gfx950.so`` (HIP kernels + C ABI, declared in
``include/llk/llk_abi.h``); this package builds it and binds it.
"""
from ._lib import LLKError, lib  # noqa: F401
from .cache import JitCache, KernelKey, WeightKey  # noqa: F401
from .decoder import (block_norm, describe_kv4_attention, kv4_attention, kv4_cache,  # noqa: F401
                      kv4_evict, kv4_evict_plan, kv4_marks, kv4_read, kv4_write)
from .ops import (PackedWeights, classify_m, describe_launch, device_info,  # noqa: F401
                  fill_normal_bf16, fused_swiglu, get_tunable, matmul, mlp, pack_device_layout,
                  select_schedule, set_schedule_db, set_tunable, swiglu_scratch_size,
                  workspace_stats, workspace_trim)
from .positions import RotaryTable, rotary  # noqa: F401
from .q4 import Q4Weights, q4_matmul, q4_quantise, q4_scratch_size, q4_swiglu  # noqa: F401

__all__ = ["JitCache", "KernelKey", "LLKError", "PackedWeights", "Q4Weights", "RotaryTable",
           "WeightKey", "block_norm", "classify_m", "describe_kv4_attention", "describe_launch",
           "device_info", "fill_normal_bf16", "fused_swiglu", "get_tunable", "kv4_attention",
           "kv4_cache", "kv4_evict", "kv4_evict_plan", "kv4_marks", "kv4_read", "kv4_write", "lib",
           "matmul", "mlp", "pack_device_layout", "q4_matmul", "q4_quantise", "q4_scratch_size",
           "q4_swiglu", "rotary", "select_schedule", "set_schedule_db", "set_tunable",
           "swiglu_scratch_size", "workspace_stats", "workspace_trim"]
