import importlib

from .fp16_fused_expert import expert_swiglu, maybe_run_fp16_fused_expert
from .grouped_expert import GroupedExperts, SharedExperts
from .qwen_topk_softmax import qwen_topk_softmax

# loaded when first asked for
_LAZY = {
    "route_experts": "expert_router",
    "quantize_rows_fp8": "fp8_blocks",
    "quantize_weight_fp8": "fp8_blocks",
    "Fp8Linear": "fp8_blocks",
    "Fp8GroupedExperts": "fp8_expert",
    "Fp8SharedExperts": "fp8_expert",
    "rotate_positions": "rotary",
    "Fp8KVCache": "fp8_cache",
}

__all__ = ["maybe_run_fp16_fused_expert", "qwen_topk_softmax", "expert_swiglu", "GroupedExperts", "SharedExperts",
           *_LAZY]


def __getattr__(name):
    if name not in _LAZY:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    value = globals()[name] = getattr(importlib.import_module(f".{_LAZY[name]}", __name__), name)
    return value
