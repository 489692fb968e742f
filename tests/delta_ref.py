"""Plain 64-bit implementations of the gated delta rule and of filtered sampling, for the op tests."""
import numpy as np


def delta_rule(q, k, v, a, b, A_log, dt_bias, S, lens, scale, norm):
    """Token by token in float64 (numpy).  q, k [N][hk][dk], v [N][hv][dv], a, b [N][hv], S [n][hv][dv][dk] (the
    sequences' starting states).  Returns o, the final states, and the sizes that rounding errors scale with:
    for o, scale |S_r| |q| of each value, for the states, the norm a head's state had or still remembers."""
    q, k, v, a, b, S = (np.asarray(x, np.float64) for x in (q, k, v, a, b, S))
    rep = v.shape[1] // q.shape[1]
    if norm:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6) for x in (q, k))
    q, k = np.repeat(q, rep, 1), np.repeat(k, rep, 1)
    alpha = np.exp(-np.exp(np.asarray(A_log, np.float64)) * np.logaddexp(0, a + dt_bias))
    with np.errstate(over="ignore"):
        beta = 1 / (1 + np.exp(-b))
    o, size, S = np.zeros(v.shape), np.zeros(v.shape), S.copy()
    held = np.sqrt((S * S).sum((-1, -2)))
    t = 0
    for i, n in enumerate(lens):
        for _ in range(n):
            D = alpha[t][:, None, None] * S[i]
            u = beta[t][:, None] * (v[t] - np.einsum("hvk,hk->hv", D, k[t]))
            S[i] = D + u[:, :, None] * k[t][:, None, :]
            o[t] = scale * np.einsum("hvk,hk->hv", S[i], q[t])
            # the state's row before and after, and what was added to it
            rows = np.maximum(np.sqrt((S[i] ** 2).sum(-1)), np.sqrt((D ** 2).sum(-1)))
            rows = np.maximum(rows, np.abs(u) * np.sqrt((k[t] ** 2).sum(-1))[:, None])
            size[t] = scale * rows * np.sqrt((q[t] ** 2).sum(-1))[:, None]
            held[i] = np.maximum(alpha[t] * held[i], np.sqrt((rows ** 2).sum(-1)))
            t += 1
    return o, S, size, held


def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seen=None, rep=1.0):
    """(token, kept, prob) of one row of fp32 logits: sorted, in float64."""
    logits = np.asarray(logits, np.float32)
    greedy = not temperature > 0
    with np.errstate(invalid="ignore", over="ignore"):
        x = logits if greedy else logits / np.float32(temperature)
        if seen is not None:
            x = np.where(seen, x / np.float32(rep), x)
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return -1, 0, 0.0
    k = 1 if greedy else top_k
    if k > 0:
        order = order[:k]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp(x[order] - top))
    stay = np.ones(len(order), bool)
    if top_p < 1:
        stay &= np.cumsum(w) - w <= max(float(np.float32(top_p)), 0.0) * w.sum()
    stay &= (w >= float(np.float32(min_p))) | (w == 1.0)
    order, w = order[stay], w[stay]
    by = np.argsort(order)
    upto = np.cumsum(w[by])
    u = min(max(float(u), 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    j = min(int((upto <= u * upto[-1]).sum()), len(by) - 1)
    return int(order[by][j]), len(order), w[by][j] / upto[-1]
