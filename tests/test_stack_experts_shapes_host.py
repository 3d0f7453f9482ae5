"""Shapes of a file's tensors on their way to nl_upload_tensor (nanollama_amd.stack): three dimensions are the experts' alone, and theirs are checked."""
import pytest

from nanollama_amd import synth_stack as ss
from nanollama_amd.designs import DESIGNS
from nanollama_amd.stack import rows_and_columns
from stack_models import config, gla, weights

CFG = config([{**gla(), "mlp": ss.routed(6, 2, 24)}, gla(ff=20)])
W = weights(CFG)
SPEC = DESIGNS["Ganidra"](CFG, lambda n: W[n].shape)


def test_every_tensor_of_a_model():
    D = CFG["width"]
    for name, source in SPEC.tensors.items():
        rows, cols = rows_and_columns(SPEC, name, source, W[source].shape)
        assert rows * cols == W[source].size and cols == W[source].shape[-1]
    at = lambda k, shape: rows_and_columns(SPEC, f"layers.0.ff.experts.{k}", "s", shape)  # noqa: E731
    assert at("gate", (6, 24, D)) == (144, D) and at("down", (6, D, 24)) == (6 * D, 24) and at("up", (144, D)) == (144, D)


@pytest.mark.parametrize("name, shape, text", [
    ("layers.0.ff.experts.gate", (24, 6, 64), "expected 6 experts"), ("layers.0.ff.experts.down", (3, 128, 24), "expected 6 experts"),
    ("layers.0.ff.experts.up", (6, 2, 12, 64), "4 dimensions"), ("layers.0.ff.router", (1, 6, 64), "3 dimensions"), ("layers.1.ff.gate", (2, 10, 64), "3 dimensions"),
    ("layers.1.lin.q", (2, 32, 64), "3 dimensions"), ("embed", (), "0 dimensions"), ("final_norm", (1, 1, 64), "3 dimensions")])
def test_refusals(name, shape, text):
    with pytest.raises(ValueError, match=f"tensor s: .*{text}"):
        rows_and_columns(SPEC, name, "s", shape)
