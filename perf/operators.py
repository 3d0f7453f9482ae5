"""The operators of a feed-forward of experts, as cases that can be timed and compared: the choice of experts (route), the experts' gated
products over ragged groups of tokens (experts), and what closes a block (residual_norm: a norm behind it, its gate and residual scale, the norm in
front of the next).

`own` chooses between the plain form (elementary torch operations in 32 bits) and nanollama_amd.ops.  Widths are those of the tiers mini (768),
goldie (1536) and wide (4096); numbers and widths of experts are generic.
"""
from __future__ import annotations

import math
import random
from typing import List

import torch

own = False

EPS = 1e-5


# ---------------------------------------------------------------- the cases

def listed() -> List[dict]:
    return [
        # one stream's next token: the smallest call, latency alone
        dict(name="route-token", op="route", n=1, experts=64, k=8, score="softmax", renorm=True, scale=1.0),
        # the decode batch of a serving host, scores by themselves and a bias that balances the load
        dict(name="route-streams", op="route", n=64, experts=96, k=6, score="sigmoid", renorm=True, scale=2.5),
        # a batch of long prompts to many small experts
        dict(name="route-prompts", op="route", n=8191, experts=256, k=8, score="sigmoid", renorm=True, scale=2.5),
        # one stream's next token: the weights of eight experts, once
        dict(name="experts-token", op="experts", n=1, dim=768, ff=512, experts=64, k=8, dtype="bfloat16"),
        # decode streams side by side: nearly every expert, a handful of tokens each
        dict(name="experts-streams", op="experts", n=64, dim=1536, ff=1024, experts=64, k=6, dtype="bfloat16"),
        # a page to few large experts; an odd number of tokens
        dict(name="experts-page", op="experts", n=333, dim=768, ff=2048, experts=8, k=2, dtype="bfloat16"),
        # the same in 32 bits, widths that fill no tile
        dict(name="experts-page-f32", op="experts", n=77, dim=760, ff=500, experts=16, k=4, dtype="float32"),
        # a document to many small experts
        dict(name="experts-document", op="experts", n=2047, dim=1536, ff=768, experts=64, k=8, dtype="bfloat16"),
        # a prompt at the largest tier's width: the largest products
        dict(name="experts-wide", op="experts", n=993, dim=4096, ff=11008, experts=8, k=2, dtype="bfloat16"),
        # what closes a block of one token
        dict(name="close-token", op="close", n=1, dim=768, dtype="bfloat16", post=True, gate="channel"),
        # of a document, a gate per channel
        dict(name="close-document", op="close", n=2047, dim=1536, dtype="bfloat16", post=True, gate="channel"),
        # of a batch of prompts at the largest width, a gate of every token's own
        dict(name="close-wide", op="close", n=8191, dim=4096, dtype="bfloat16", post=True, gate="token"),
    ]


def _spread(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random) -> dict:
    """A token to a batch of prompts; few large experts to many small ones; widths in whole 16-byte pieces for the products, any for the rest."""
    op = rng.choice(["route", "experts", "experts", "experts", "close"])
    if op == "route":
        experts = _spread(rng, 4, 384)
        return dict(op=op, n=_spread(rng, 1, 8191), experts=experts, k=rng.randint(1, min(12, experts)), score=rng.choice(["softmax", "sigmoid"]),
                    renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]))
    if op == "close":
        return dict(op=op, n=_spread(rng, 1, 8191), dim=_spread(rng, 100, 4096), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]),
                    post=rng.random() < 0.7, gate=rng.choice(["none", "channel", "token"]))
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    case = dict(op=op, n=_spread(rng, 1, 2047), dim=8 * rng.randint(16, 256), ff=8 * rng.randint(8, 256), experts=_spread(rng, 4, 96), k=1, dtype=dtype)
    case["k"] = rng.randint(1, min(8, case["experts"]))
    most = 4e10 if dtype == "float32" else 4e11
    while case["n"] > 1 and work(case)["flops"] > most:
        case["n"] = case["n"] * 3 // 4
    while work(case)["bytes"] > 2e9:
        case["experts"] = max(case["k"], case["experts"] * 3 // 4)
    return case


# ---------------------------------------------------------------- inputs

def _type(case):
    return torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    normal = lambda *size: torch.randn(*size, generator=g, device="cuda")  # noqa: E731
    n = case["n"]
    if case["op"] == "route":
        E = case["experts"]
        # experts differ in how often they are asked for; the bias pulls the other way
        liking = normal(E)
        return dict(case=case, logits=normal(n, E) + 0.7 * liking, bias=-0.1 * liking if case["score"] == "sigmoid" else None,
                    ids=torch.empty(n, case["k"], dtype=torch.int32, device="cuda"), weights=torch.empty(n, case["k"], device="cuda"))
    T, D = _type(case), case["dim"]
    if case["op"] == "close":
        gate = None if case["gate"] == "none" else 1 + 0.2 * normal(D) if case["gate"] == "channel" else torch.sigmoid(normal(n, D))
        return dict(case=case, x=normal(n, D), d=(0.5 * normal(n, D)).to(T), post=1 + 0.1 * normal(D) if case["post"] else None, gate=gate, scale=0.7,
                    pre=1 + 0.1 * normal(D), x_out=torch.empty(n, D, device="cuda"), h=torch.empty(n, D, dtype=T, device="cuda"))
    E, F, k = case["experts"], case["ff"], case["k"]
    logits = normal(n, E) + 0.5 * normal(E)
    top = torch.softmax(logits, 1).topk(k, 1)
    matrix = lambda rows, cols: torch.empty(E, rows, cols, dtype=T, device="cuda").normal_(0, cols ** -0.5, generator=g)  # noqa: E731
    return dict(case=case, x=normal(n, D).to(T), ids=top.indices.to(torch.int32), weights=(top.values / top.values.sum(1, keepdim=True)).contiguous(),
                gate=matrix(F, D), up=matrix(F, D), down=matrix(D, F), y=torch.empty(n, D, dtype=T, device="cuda"))


# ---------------------------------------------------------------- the framework's operators

def _run_own(s: dict):
    from nanollama_amd import ops
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "route":
        ops.route(s["logits"], s["ids"], s["weights"], score=case["score"], bias=s["bias"], renorm=case["renorm"], scale=case["scale"], stream=stream)
        return dict(ids=s["ids"], weights=s["weights"])
    if case["op"] == "close":
        ops.residual_norm(s["x"], s["d"], s["x_out"], s["h"], pre=s["pre"], post=s["post"], gate=s["gate"], scale=s["scale"], eps=EPS, stream=stream)
        return dict(x=s["x_out"], h=s["h"])
    if "workspace" not in s:
        s["workspace"] = torch.empty(ops.experts_workspace(case["n"], case["k"], case["experts"], case["dim"], case["ff"], case["dtype"]), dtype=torch.uint8, device="cuda")
    ops.experts(s["x"], s["ids"], s["weights"], s["gate"], s["up"], s["down"], s["y"], s["workspace"], act="silu", stream=stream)
    return dict(y=s["y"])


# ---------------------------------------------------------------- the plain forms

def _route(s: dict):
    case, l = s["case"], s["logits"].double()          # (keys next to each other decide: 64 bits)
    score = torch.softmax(l, 1) if case["score"] == "softmax" else 1 / (1 + torch.exp(-l))
    key = l if s["bias"] is None else score + s["bias"].double()
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :case["k"]]
    w = score.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return dict(ids=ids.to(torch.int32), weights=(w * case["scale"]).float())


def _close(s: dict):
    v = s["d"].float()
    if s["post"] is not None:
        v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * s["post"]
    if s["gate"] is not None:
        v = v * s["gate"]
    x = s["x"] + s["scale"] * v
    return dict(x=x, h=(x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["pre"]).to(s["d"].dtype))


def _experts(s: dict):
    k, x, E = s["case"]["k"], s["x"].float(), s["gate"].shape[0]
    slot = torch.argsort(s["ids"].reshape(-1), stable=True)        # tokens by expert
    counts = torch.bincount(s["ids"].reshape(-1).long(), minlength=E).tolist()
    y, at = torch.zeros_like(x), 0
    for e, m in enumerate(counts):
        if m:
            mine = slot[at:at + m]
            rows = x[mine // k]
            a, b = rows @ s["gate"][e].float().T, rows @ s["up"][e].float().T
            h = a / (1 + torch.exp(-a)) * b
            y.index_add_(0, mine // k, h @ s["down"][e].float().T * s["weights"].reshape(-1)[mine, None])
            at += m
    return dict(y=y.to(s["x"].dtype))


def run(state: dict):
    if own:
        return _run_own(state)
    return {"route": _route, "close": _close, "experts": _experts}[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case: dict) -> dict:
    n = case["n"]
    if case["op"] == "route":
        return dict(bytes=4 * n * case["experts"] + 8 * n * case["k"], flops=4 * n * case["experts"])
    D, size = case["dim"], 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "close":
        return dict(bytes=n * D * (8 + 2 * size + (4 if case["gate"] == "token" else 0)) + 12 * D, flops=10 * n * D)
    E, k, F = case["experts"], case["k"], case["ff"]
    hit = E * (1 - (1 - k / E) ** n)                    # experts that some token chose, as expected
    return dict(bytes=int(3 * hit * D * F * size + 2 * n * D * size + 8 * n * k), flops=6 * n * k * D * F)


# ---------------------------------------------------------------- from the definition, in 64 bits

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "route":
        l = s["logits"].double()
        p = torch.sigmoid(l) if case["score"] == "sigmoid" else torch.exp(l - torch.logsumexp(l, 1, keepdim=True))
        chosen = torch.zeros_like(p, dtype=torch.bool)
        left = p + s["bias"].double() if s["bias"] is not None else l.clone()
        w = []
        for _ in range(case["k"]):                      # the largest that is left, k times
            best = left.argmax(1, keepdim=True)
            w.append(p.gather(1, best))
            chosen.scatter_(1, best, True)
            left = left.masked_fill(chosen, -math.inf)
        w = torch.cat(w, 1)
        total = (p * chosen).sum(1, keepdim=True) if case["renorm"] else 1.0
        return dict(ids=None, weights=case["scale"] * w / total)
    if case["op"] == "close":
        rms = lambda v: v / torch.sqrt(v.square().sum(1, keepdim=True) / v.shape[1] + EPS)  # noqa: E731
        v = s["d"].double()
        v = rms(v) * s["post"].double() if s["post"] is not None else v
        x = s["x"].double() + s["scale"] * (v if s["gate"] is None else v * s["gate"].double())
        return dict(x=x, h=rms(x) * s["pre"].double())
    # the weight that every token gives to every expert; the experts one by one over the tokens that give any
    coef = torch.zeros(case["n"], case["experts"], dtype=torch.float64, device="cuda").scatter_add_(1, s["ids"].long(), s["weights"].double())
    y = torch.zeros(case["n"], case["dim"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        t = coef[:, e].nonzero()[:, 0]
        if t.numel():
            x = s["x"][t].double()
            z = torch.nn.functional.linear(x, s["gate"][e].double())
            y[t] += coef[t, e, None] * torch.nn.functional.linear(z * torch.sigmoid(z) * torch.nn.functional.linear(x, s["up"][e].double()), s["down"][e].double())
    return dict(y=y)
