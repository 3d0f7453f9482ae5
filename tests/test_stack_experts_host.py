"""Layer-stack models with experts without a GPU: what a design reads, what it refuses, and the oracle's experts."""
import copy

import numpy as np
import pytest

from nanollama_amd import _lib, registry
from nanollama_amd import synth_stack as ss
from nanollama_amd.designs import DESIGNS
from nanollama_amd.stack import Experts, StackConfig
from oracle import stack_oracle as so
from stack_models import config, floats, gla, lat, lconfig, par, weights


def routed(layer, *args, **more):
    return {**layer, "mlp": ss.routed(*args, **more)}


CASES = [config([routed(gla(), 12, 3, 48), par(ff=20), routed(par(), 9, 4, 40, score="sigmoid", renorm=False, scale=2.5, bias=True)]),
         lconfig([routed(lat(), 8, 2, 40), lat(ff=32), routed(lat(2), 6, 1, 24, score="sigmoid", bias=True)])]


@pytest.mark.parametrize("cfg", CASES, ids=lambda c: c["architecture"])
def test_every_tensor_has_its_place(cfg):
    w = weights(cfg)
    s = DESIGNS[cfg["architecture"]](cfg, lambda n: w[n].shape)
    assert sorted(s.tensors.values()) == sorted(w)
    act = "gelu_tanh" if cfg["architecture"] == "Ganidra" else "silu"
    for layer, entry in zip(s.layers, cfg["layers"]):
        m = entry["mlp"]
        if m and m["kind"] == "routed":
            assert layer.ff == 0 and layer.experts == Experts(m["experts"], m["per_token"], m["ff"], act, m.get("score", "softmax"), m.get("renorm", True),
                                                              m.get("bias", False), m.get("scale", 1.0))
        else:
            assert layer.experts is None
    assert w["l0.mlp.experts.gate"].shape == (cfg["layers"][0]["mlp"]["experts"], cfg["layers"][0]["mlp"]["ff"], cfg["width"])
    assert StackConfig(s, 64, "bfloat16", 1).interm_size >= 48


@pytest.mark.parametrize("cfg", CASES, ids=lambda c: c["architecture"])
def test_folders_and_refusals(cfg, tmp_path):
    w = weights(cfg)
    assert registry.read_spec(ss.write_folder(str(tmp_path / "a"), cfg, w)) is not None
    bad = copy.deepcopy(cfg)
    bad["layers"][0]["mlp"]["score"] = "tanh"
    with pytest.raises(ValueError, match="unknown score"):
        DESIGNS[cfg["architecture"]](bad, lambda n: w[n].shape)


def test_no_handle():
    assert _lib.stack_lib().nl_stack_experts(None, 0, None) == -1


def test_experts_that_are_alike_are_one_feed_forward():
    """With equal experts and weights that sum to one the oracle's experts are the dense feed-forward, whatever is chosen."""
    cfg = config([routed(gla(), 6, 2, 24)])
    w = floats(weights(cfg))
    for k in ("gate", "up", "down"):
        w[f"l0.mlp.experts.{k}"][:] = w[f"l0.mlp.experts.{k}"][0]
        w[f"l0.mlp.{k}"] = w[f"l0.mlp.experts.{k}"][0]
    dense = copy.deepcopy(cfg)
    dense["layers"][0]["mlp"] = {"kind": "dense", "ff": 24}
    ids = list(range(11))
    assert np.allclose(so.forward(cfg, w, ids), so.forward(dense, w, ids), rtol=1e-12, atol=1e-12)
