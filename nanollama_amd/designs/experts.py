"""The feed-forward of experts that a layer of either design may have: {"kind": "routed", "experts", "per_token", "ff", "score": "softmax" or
"sigmoid", "renorm", "scale", "bias"} (the last four may be left out), tensors mlp.router [experts, width], mlp.router.b with bias,
mlp.experts.gate and up [experts, ff, width], mlp.experts.down [experts, width, ff]."""
from __future__ import annotations

from ..stack import SCORES, Experts


def routed_experts(i: int, mlp: dict, act: str, tensors: dict) -> Experts:
    score = mlp.get("score", "softmax")
    if score not in SCORES:
        raise ValueError(f"layer {i}: unknown score {score!r}")
    x = Experts(mlp["experts"], mlp["per_token"], mlp["ff"], act, score, mlp.get("renorm", True), mlp.get("bias", False), mlp.get("scale", 1.0))
    tensors[f"layers.{i}.ff.router"] = f"l{i}.mlp.router"
    if x.bias:
        tensors[f"layers.{i}.ff.router_bias"] = f"l{i}.mlp.router.b"
    tensors.update({f"layers.{i}.ff.experts.{k}": f"l{i}.mlp.experts.{k}" for k in ("gate", "up", "down")})
    return x
