"""Layer-stack models whose feed-forwards are experts, on the GPU against the float64 oracle (oracle/stack_oracle.py)."""
import ctypes as C

import numpy as np
import pytest

from nanollama_amd import _lib
from nanollama_amd import synth_stack as ss
from oracle import stack_oracle as so
from stack_models import BF16_TOL, F32_TOL, config, floats, gla, lat, lconfig, load, par, rel, tokens, weights

pytestmark = pytest.mark.gpu
TOL = {"float32": F32_TOL, "bfloat16": BF16_TOL}


def routed(layer, *args, **more):
    return {**layer, "mlp": ss.routed(*args, **more)}


# (bfloat16 only where every expert is chosen: a choice may tip on a rounding of the router's operand)
MODELS = {
    "softmax": (config([routed(gla(), 12, 3, 48), par()]), ["float32"]),
    "sigmoid_and_bias": (config([routed(par(), 9, 4, 40, score="sigmoid", renorm=False, scale=2.5, bias=True), routed(gla(), 9, 2, 40, score="sigmoid", bias=True)]), ["float32"]),
    "not_renormalised": (config([routed(gla(), 7, 2, 32, renorm=False)]), ["float32"]),
    "all_of_them": (config([routed(gla(), 5, 5, 32), gla(ff=24), routed(par(), 3, 3, 56, score="sigmoid", bias=True)]), ["float32", "bfloat16"]),
    "one_expert": (config([routed(gla(), 1, 1, 32)]), ["float32", "bfloat16"]),
    "odd_sizes": (config([routed(gla(), 5, 2, 21), routed(par(), 4, 4, 9)], vocab=77, width=50), ["float32"]),
    "odd_sizes_all": (config([routed(gla(), 4, 4, 21)], vocab=77, width=50), ["float32", "bfloat16"]),
    "loop": (config([gla(), routed(gla(), 6, 2, 32), routed(par(), 6, 3, 24)], loop=(1, 3, 3)), ["float32"]),
    "norms_behind": (lconfig([routed(lat(), 8, 2, 40), lat(ff=32), routed(lat(3), 6, 6, 24, score="sigmoid", bias=True)]), ["float32"]),
    "norms_behind_all": (lconfig([routed(lat(), 4, 4, 40), lat(ff=32)]), ["float32", "bfloat16"]),
    "many_small": (config([routed(gla(), 160, 12, 16)], width=128), ["float32"]),
}


def by_token(m, ids, stream=0):
    rows = []
    for i, t in enumerate(ids):
        m.forward(t, i, stream)
        rows.append(m.state.logits.copy())
    return np.array(rows)


@pytest.mark.parametrize("name, dtype", [(n, d) for n, (_, ds) in MODELS.items() for d in ds])
def test_prompts_and_single_tokens(name, dtype):
    cfg, _ = MODELS[name]
    w = weights(cfg, 3)
    ids = tokens(70, cfg["vocab"], seed=5)
    want, layers = so.forward(cfg, floats(w), ids, want_layers=True)
    m = load(cfg, w, dtype)
    m.trace_layers(True)
    got = m.step([(0, ids, 0, list(range(len(ids))))])[0]
    seen = m.layer_trace(len(ids))
    m.trace_layers(False)
    for r in range(len(layers)):
        assert rel(seen[r], layers[r]) < TOL[dtype], r
    assert rel(got, want) < TOL[dtype]
    assert rel(by_token(m, ids, 1), want) < TOL[dtype]
    # the same prompt in pieces and as one entry of a ragged batch
    rows = m.step([(2, ids[:33], 0, list(range(33))), (3, ids, 0, [69])])
    rows += m.step([(2, ids[33:], 33, list(range(37)))])
    assert rel(np.concatenate([rows[0], rows[2]]), want) < TOL[dtype] and rel(rows[1], want[69:]) < TOL[dtype]
    m.close()


def test_long_prompts_are_cut():
    cfg = config([routed(gla(), 8, 2, 64), routed(par(), 4, 2, 64)])
    w = weights(cfg, 8)
    ids = tokens(333, seed=6)
    want = so.forward(cfg, floats(w), ids)
    for cut in (64, 0):
        m = load(cfg, w, max_step_tokens=cut)
        m.prefill(ids)
        assert rel(m.state.logits, want[-1:]) < F32_TOL
        m.close()


@pytest.mark.parametrize("streams", [1, 3, 17, 40])
def test_decode_batches(streams):
    cfg = config([routed(gla(), 24, 4, 32), routed(par(), 6, 2, 40, score="sigmoid", bias=True)])
    w = weights(cfg, 4)
    ids = [tokens(6, seed=s) for s in range(streams)]
    m = load(cfg, w, max_streams=streams)
    for i in range(6):
        got = m.forward_batch(list(range(streams)), [t[i] for t in ids], [i] * streams, want_logits=True)
    want = np.array([so.forward(cfg, floats(w), t)[-1] for t in ids])
    logits = got[1] if isinstance(got, tuple) else got
    assert rel(logits, want) < F32_TOL
    m.close()


def test_chained_greedy_steps():
    cfg = config([routed(gla(), 16, 2, 32), routed(par(), 16, 3, 32)], loop=(0, 2, 2))
    w = weights(cfg, 9)
    prompt = tokens(9, seed=1)
    want = so.greedy(cfg, floats(w), prompt, 40)
    for flags in (0, 1):                                  # replayed graphs, and launch by launch
        m = load(cfg, w, flags=flags)
        for _ in range(2):
            m.prefill(prompt)
            first = int(np.argmax(m.state.logits))
            assert [first] + [int(t) for t in m.decode_greedy(first, len(prompt), 39)] == want
            m.reset()
        m.close()


def test_refusals():
    L = _lib.stack_lib()
    cfg = _lib.NlStackConfig(32, 64, 2, 0, 0, 1, 64, 1, 0, 0, 1, 0, 0, 0, 0, 1e-5, 1.0)
    layers = (_lib.NlLayerDesc * 2)()
    for i, d in enumerate(layers):
        d.lin = _lib.NlLinattnDesc(2, 16, 16, 4, 8.0, 1.0)
        d.ff = 32 * i
    h = C.c_void_p()
    assert L.nl_create_stack(C.byref(cfg), layers, C.byref(h)) == 0
    call = lambda layer, *a: (L.nl_stack_experts(h, layer, C.byref(_lib.NlStackExpertsDesc(*a))), L.nl_last_error(h).decode())  # noqa: E731
    good = (8, 2, 32, 1, 0, 1, 0, 1.0)
    for layer, desc, code, text in [
            (-1, good, -1, "out of range"), (2, good, -1, "out of range"), (1, good, -2, "beside a feed-forward"), (0, (0,) + good[1:], -1, "of 0 experts"),
            (0, (1025,) + good[1:], -1, "of 1025 experts"), (0, (8, 9) + good[2:], -1, "9 of 8"), (0, (64, 33) + good[2:], -1, "33 of 64"), (0, (8, 0) + good[2:], -1, "0 of 8"),
            (0, (8, 2, 0) + good[3:], -1, "width"), (0, (8, 2, 32, 5) + good[4:], -1, "activation"), (0, (8, 2, 32, 1, 3, 1, 0, 1.0), -1, "scores"),
            (0, (8, 2, 32, 1, 0, 1, 0, float("nan")), -1, "scores"), (0, (8, 2, 32, 1, 0, 1, 1, 1.0), -2, "bias")]:
        rc, message = call(layer, *desc)
        assert rc == code and text in message, (desc, rc, message)
    assert L.nl_stack_experts(h, 0, None) == -1
    assert call(0, *good)[0] == 0
    rc, message = call(0, *good)
    assert rc < 0 and "already" in message
    x = np.zeros((8 * 32, 64), np.float32)
    up = lambda name, rows, cols: L.nl_upload_tensor(h, name, 0, x.ctypes.data, rows * cols * 4, rows, cols)  # noqa: E731
    assert up(b"layers.0.ff.experts.gate", 8 * 32, 64) == 0 and up(b"layers.0.ff.experts.down", 8 * 64, 32) == 0
    assert up(b"layers.0.ff.experts.gate", 64, 8 * 32) == -1 and up(b"layers.0.ff.gate", 32, 64) == -1 and up(b"layers.0.ff.router_bias", 1, 8) == -1
    assert up(b"layers.1.ff.router", 8, 64) == -1
    assert L.nl_finalize(h) < 0 and b"not uploaded" in L.nl_last_error(h)
    L.nl_destroy(h)


@pytest.mark.parametrize("cfg", [MODELS["sigmoid_and_bias"][0], MODELS["norms_behind"][0]], ids=["Ganidra", "Pabalix"])
def test_from_a_folder_through_the_scheduler(cfg, tmp_path):
    from nanollama_amd import registry
    from nanollama_amd.scheduler import Scheduler
    w = weights(cfg, 6)
    m = registry.load_model(ss.write_folder(str(tmp_path / "model"), cfg, w), max_streams=3, dtype="float32", seq_len=128)
    prompts = [tokens(n, cfg["vocab"], seed=n) for n in (3, 17, 1, 40, 9)]
    got = Scheduler(m).generate(prompts, 8)
    want = [so.greedy(cfg, floats(w), p, 8) for p in prompts]
    assert [[int(t) for t in g] for g in got] == want
    m.close()
