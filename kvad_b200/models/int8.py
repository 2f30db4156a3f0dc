"""A plan in 8 bits: the same layers, weights and run order, with the parts that hold weights, activations and cache in 8-bit codes.

Every block has to be a `pre_norm` one of plain causal attention and a dense feed-forward (GPT-2's); the embedding and the head stay as they
are.  Which tensors a checkpoint has to have does not change.
"""
from __future__ import annotations

from dataclasses import replace

from ..parts.base import PartSpec
from .plan import ModelPlan


def int8_plan(plan: ModelPlan) -> ModelPlan:
    blocks = []
    for spec in plan.blocks:
        mixer, ff = spec.params.get("mixer"), spec.params.get("feed_forward")
        if spec.kind != "pre_norm" or mixer.kind != "causal_attention" or ff.kind != "dense_mlp":
            raise ValueError(f"no 8-bit form of `{plan.arch_id}`: its blocks are not pre-norm blocks of plain causal attention and a dense feed-forward")
        blocks.append(PartSpec("pre_norm_int8", {**spec.params, "mixer": PartSpec("causal_attention_int8", mixer.params),
                                                 "feed_forward": PartSpec("dense_mlp_int8", ff.params)}))
    return replace(plan, blocks=tuple(blocks), summary=plan.summary + " \u00b7 8-bit products and cache" if plan.summary else plan.summary)
