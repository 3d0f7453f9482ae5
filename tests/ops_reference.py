"""The operators of nanollama_amd.ops in 64 bits (numpy), and how far 32- and 16-bit arithmetic may be from that: every rounding is at most half a
step of its type, a sum of n terms in 32 bits at most n of them relative to the sum of the terms' sizes."""
import numpy as np

U32, U16 = 2.0 ** -24, 2.0 ** -8          # half a step: float32, bfloat16


def sigmoid(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z))


def act(name, z):
    return z * sigmoid(z) if name == "silu" else z * sigmoid(2.0 * np.sqrt(2.0 / np.pi) * (z + 0.044715 * z ** 3))


def route(logits, k, score="softmax", bias=None, renorm=True, scale=1.0):
    """ids, weights, and the weights' bound."""
    n, E = logits.shape
    ids, w = np.full((n, k), -1, np.int32), np.zeros((n, k))
    bound = np.zeros((n, k))
    for t in range(n):
        l = logits[t].astype(np.float64)
        live = [e for e in range(E) if l[e] > -np.inf and (bias is None or bias[e] > -np.inf)]
        if not live:
            continue
        m = max(l[live])
        with np.errstate(invalid="ignore"):
            s = np.array([sigmoid(l[e]) if score == "sigmoid" else 1.0 if l[e] == m else np.exp(l[e] - m) for e in live])
        key = l[live] if bias is None else s + bias[live].astype(np.float64)
        order = np.lexsort((live, -key))[:k]
        at = l[live][order]
        ids[t, :len(order)] = np.array(live)[order]
        if score == "sigmoid" and renorm:                # shares of sigmoids, from their logarithms
            top = max(at)
            log = -np.logaddexp(0.0, -at) if top < np.inf else np.log(s[order])
            chosen = np.exp(log - max(log))
        else:
            chosen = s[order]
        total = chosen.sum() if renorm else 1.0 if score == "sigmoid" else s.sum()
        w[t, :len(order)] = scale * chosen / total
        # exp of a rounded difference: half a step of it; exp, reciprocal and quotient: 16 half steps; the sum of E such terms
        top = m if score == "softmax" else max(at)
        far = np.minimum(np.abs(np.where(at == top, 0.0, at - (top if top < np.inf else 0.0))), 110.0)
        bound[t, :len(order)] = np.abs(w[t, :len(order)]) * (far + 18 + E) * U32 + abs(scale) * 2.0 ** -126
    return ids, w, bound


def experts(x, ids, weights, gate, up, down, name="silu", half=U32):
    """y and a bound for every element of it; half: half a step of the arrays' type (inputs are that type's numbers)."""
    x, gate, up, down, w = (np.asarray(a, np.float64) for a in (x, gate, up, down, weights))
    (n, D), (E, F, _) = x.shape, gate.shape
    y, bound = np.zeros((n, D)), np.zeros((n, D))
    size = np.zeros((n, D))
    for e in range(E):
        t, j = np.nonzero(ids == e)
        if not len(t):
            continue
        g, u = x[t] @ gate[e].T, x[t] @ up[e].T
        dg, du = (D + 2) * U32 * (np.abs(x[t]) @ np.abs(gate[e]).T), (D + 2) * U32 * (np.abs(x[t]) @ np.abs(up[e]).T)
        h = act(name, g) * u
        # |act'| <= 1.13; the activation's own functions: 16 steps of 32 bits (|z| <= 100); h is rounded to the type
        dh = 1.13 * dg * np.abs(u) + (np.abs(act(name, g)) + 1.13 * dg) * du + np.abs(h) * 32 * U32
        dh += (half if half > U32 else U32) * (np.abs(h) + dh)
        p, sp = h @ down[e].T, np.abs(h) @ np.abs(down[e]).T
        dp = dh @ np.abs(down[e]).T + (F + 2) * U32 * (sp + dh @ np.abs(down[e]).T)
        c = w[t, j][:, None]
        part, dpart = c * p, np.abs(c) * dp
        dpart += 2 * U32 * (np.abs(part) + dpart)                          # weighted
        np.add.at(y, t, part)
        np.add.at(bound, t, dpart)
        np.add.at(size, t, np.abs(part) + dpart)
    bound += ids.shape[1] * U32 * size
    return y, bound + half * (np.abs(y) + bound) + 2.0 ** -133


def residual_norm(x, d, pre, post=None, gate=None, scale=1.0, eps=1e-5, half=U32):
    """x_out, h and their bounds."""
    x, d = np.asarray(x, np.float64), np.asarray(d, np.float64)
    D = x.shape[1]
    rms = lambda v: v / np.sqrt(np.mean(v * v, -1, keepdims=True) + eps)  # noqa: E731
    v = d if post is None else rms(d) * np.asarray(post, np.float64)
    if gate is not None:
        v = v * np.asarray(gate, np.float64)
    # the mean's sum, root and reciprocal (D / 2 + 4 roundings of the norm), the factors
    dv = np.abs(v) * (D / 2 + 10) * U32
    xo = x + scale * v
    dx = abs(scale) * dv + 3 * U32 * (np.abs(x) + abs(scale) * np.abs(v))
    h = rms(xo) * np.asarray(pre, np.float64)
    r = np.sqrt(np.mean(xo * xo, -1, keepdims=True) + eps)
    dh = np.abs(np.asarray(pre, np.float64)) / r * dx + np.abs(h) * (np.sqrt(np.mean(dx * dx, -1, keepdims=True)) / r + (D / 2 + 10) * U32)
    return xo, h, dx + 2.0 ** -140, dh + half * (np.abs(h) + dh) + 2.0 ** -133
