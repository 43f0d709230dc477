"""Router of grouped experts with a balancing bias, beside ``qwen_topk_softmax``.

``route_experts`` covers what routers of larger MoE layers add to a softmax
top-k: sigmoid scores, a bias that takes part in the choice and not in the
weights, groups of experts of which the best stay, a final scale.  One
tm_route_experts call; keys are compared in 64 bits, ties go to the lower id.
"""

from __future__ import annotations

import torch

from .. import _native as N

_SCORING = {"softmax": N.TM_ROUTE_SOFTMAX, "sigmoid": N.TM_ROUTE_SIGMOID}
_GROUP_RULE = {"max": N.TM_GROUP_MAX, "top2": N.TM_GROUP_TOP2}


def route_experts(router_logits: torch.Tensor, top_k: int, *, scoring: str = "softmax",
                  bias: torch.Tensor | None = None, n_groups: int = 1, topk_groups: int | None = None,
                  group_rule: str = "max", normalize_topk: bool = False, scale: float = 1.0):
    """(weights fp32, ids int64), [N, top_k] each, for ``router_logits`` [N, E]
    (float32, float16 or bfloat16, unit stride along E or copied).

    scoring: "softmax" or "sigmoid" scores s.  bias [E]: experts are chosen by
    s + bias, weighted by s.  n_groups > 1: only experts of the ``topk_groups``
    (default: all) best groups are chosen, a group being worth its best key
    ("max") or the sum of its two best ("top2").  normalize_topk divides the
    weights by their sum; scale multiplies them.  An expert whose logit (or
    bias) is -inf or NaN is chosen after every other one, with weight 0.

    HybridStorageManager.combine_slots(target="orig_sum") takes the weights as they
    are; GlobalTable.gather_combine (and the layer calls, which run a softmax router
    of their own) divides them by their sum, so neither scale nor unnormalised
    weights reach its output."""
    if router_logits.dim() != 2:
        raise ValueError(f"route_experts expects 2D logits, got {tuple(router_logits.shape)}")
    if scoring not in _SCORING or group_rule not in _GROUP_RULE:
        raise ValueError(f"route_experts: scoring {scoring!r} / group_rule {group_rule!r}; expected one of "
                         f"{sorted(_SCORING)} / {sorted(_GROUP_RULE)}")
    dev = N.require_hip(router_logits, bias)
    tag = N.dtype_tag(router_logits.dtype)
    n, n_exp = router_logits.shape
    logits = router_logits
    if (logits.stride(1) != 1 and n_exp > 1) or (logits.stride(0) < n_exp and n > 1):  # (stride 0: one row for all)
        logits = logits.contiguous()
    if bias is not None:
        if bias.shape != (n_exp,):
            raise ValueError(f"route_experts: bias must be [{n_exp}], got {tuple(bias.shape)}")
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.to(torch.float32).contiguous()
    weights = torch.empty((n, top_k), dtype=torch.float32, device=dev)
    ids = torch.empty((n, top_k), dtype=torch.long, device=dev)
    with N.on_device(dev):
        N.call("tm_route_experts", tag, N.ptr(logits), n, n_exp, max(logits.stride(0), n_exp), N.ptr(bias),
               _SCORING[scoring], int(n_groups), int(n_groups if topk_groups is None else topk_groups),
               _GROUP_RULE[group_rule], int(top_k), 1 if normalize_topk else 0, float(scale), N.ptr(weights),
               N.ptr(ids), N.stream(dev))
    return weights, ids
