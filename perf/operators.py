"""Cases, plain forms and 64-bit definitions of the gated delta rule and of filtered sampling.

Three operators of a recurrent decode engine, each next to one that the engine offers already:

  step     one token of every running sequence through the gated delta rule: the per-slot state S is decayed,
           corrected along the key and read along the query (beside the Mamba-2 state update of one token)
  prefill  the same recurrence over ragged prompts, from and into the slots' states (beside the prompt scan)
  sample   the choice of the next token from logits, with a temperature, top-k, top-p and min-p of its own for
           every row and given uniform numbers (beside the sampling epilogue)

With q, k of head h (optionally scaled to unit length), g = -exp(A_log) softplus(a + dt_bias), beta = sigmoid(b):

  S <- e^g S + beta (v - e^g S k) k^T,      o = scale * S q,      S [dv][dk] in fp32
"""
import math
import random

import numpy as np
import torch

own = False

#: (key heads, value heads, key width, value width): heads that share one key as the engine's 1.3B and 2.7B
#: shapes share B and C, grouped heads, one key head per value head, and narrow ones.
HEADS = ((1, 64, 128, 64), (1, 80, 128, 64), (16, 32, 128, 128), (8, 8, 64, 64), (4, 12, 128, 48), (6, 6, 128, 128))
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CHUNK = 64
EPS = 1e-6


def listed():
    def delta(op, name, heads, kind, norm=True, **more):
        hk, hv, dk, dv = heads
        if op == "prefill":
            more.setdefault("even", False)
        return {"op": op, "name": name, "hk": hk, "hv": hv, "dk": dk, "dv": dv, "type": kind, "norm": norm, **more}

    return [
        # one sequence being decoded: latency is all that counts
        delta("step", "step-1", HEADS[0], "fp16", rows=1, slots=1),
        # a serving batch of 32 on grouped heads, sequences scattered over more slots than rows
        delta("step", "step-32", HEADS[2], "bf16", rows=32, slots=48),
        # the largest decode batch of the 1.3B shape
        delta("step", "step-256", HEADS[0], "fp16", rows=256, slots=256),
        # one 16-token prompt, the shortest the engine's own workload has
        delta("prefill", "prefill-16", HEADS[0], "fp16", tokens=16, seqs=1),
        # prompts of a few dozen tokens admitted together, some of one token, one empty
        delta("prefill", "prefill-short", HEADS[3], "bf16", norm=False, tokens=777, seqs=19),
        # a ragged admission of long and short prompts
        delta("prefill", "prefill-ragged", HEADS[2], "bf16", tokens=16384, seqs=24),
        # a long document in one sequence: the recurrence itself is the longest chain
        delta("prefill", "prefill-long", HEADS[2], "fp16", tokens=32768, seqs=1),
        # a batch of 64-token prompts of the 1.3B shape
        delta("prefill", "prefill-64x64", HEADS[0], "fp16", tokens=4096, seqs=64, even=True),
        # one row: the end of a batch-1 step
        {"op": "sample", "name": "sample-1", "rows": 1, "vocab": 50280, "type": "fp32", "mix": "all"},
        # a serving batch whose requests all differ in their settings, some under a token mask
        {"op": "sample", "name": "sample-32", "rows": 32, "vocab": 50280, "type": "fp32", "mix": "masked"},
        # a batch on a vocabulary of odd size in 16 bits, where equal logits are common
        {"op": "sample", "name": "sample-wide", "rows": 48, "vocab": 151937, "type": "bf16", "mix": "nucleus"},
        # the largest batch of the engine's own vocabulary
        {"op": "sample", "name": "sample-256", "rows": 256, "vocab": 50280, "type": "fp32", "mix": "all"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("step", "prefill", "sample"))
    if op == "sample":
        vocab = _log(rng, 500, 160000)
        return {"op": op, "rows": _log(rng, 1, max(1, min(256, 256 * 50280 // vocab))), "vocab": vocab,
                "type": rng.choice(("fp32", "fp32", "bf16", "fp16")), "mix": rng.choice(("all", "masked", "nucleus", "topk"))}
    hk, hv, dk, dv = rng.choice(HEADS)
    c = {"op": op, "hk": hk, "hv": hv, "dk": dk, "dv": dv, "type": rng.choice(("fp16", "bf16")), "norm": rng.random() < 0.8}
    if op == "step":
        rows = _log(rng, 1, 204 if hv == 80 else 256)
        return {**c, "rows": rows, "slots": rows + rng.choice((0, 0, rows // 2))}
    tokens = _log(rng, 1, 32768)
    if hv > 32:
        tokens = min(tokens, 16384)
    return {**c, "tokens": tokens, "seqs": min(max(1, tokens // 4), _log(rng, 1, 64)), "even": rng.random() < 0.3}


# ------------------------------------------------------------------------------------------------ inputs


def _lengths(case, seed):
    """Lengths that add up to case["tokens"]: all alike, or one in eight empty or of one token and the others spread widely."""
    n, total = case["seqs"], case["tokens"]
    if case["even"]:
        return [total // n + (i < total % n) for i in range(n)]
    rng = random.Random("%d lengths of %d, %d" % (n, total, seed))
    cut = [i for i in range(n) if n > 1 and rng.random() < 0.125]
    weight = [0.0 if i in cut else math.exp(rng.gauss(0, 1)) for i in range(n)]
    if sum(weight) == 0:
        weight[0] = 1.0
    lens = [int(total * w / sum(weight)) for w in weight]
    for j, i in enumerate(cut):
        lens[i] = min(j % 2, total)
    while sum(lens) > total:
        lens[lens.index(max(lens))] -= 1
    lens[lens.index(max(lens))] += total - sum(lens)
    return lens


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=gen, dtype=dtype)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    t = TYPES[case["type"]]
    if case["op"] == "sample":
        B, V = case["rows"], case["vocab"]
        # logits of a trained model: a broad bulk and a few tokens far above it, sharper in some rows
        logits = randn(B, V) * (1.0 + 2.0 * rand(B, 1))
        logits += 9.0 * (rand(B, V) < 20.0 / V) * rand(B, V)
        if case["mix"] == "masked":
            logits = logits.masked_fill(rand(B, V) < rand(B, 1), -math.inf)
        temperature = 0.3 + 1.2 * rand(B)
        top_k = torch.exp(rand(B) * math.log(min(V, 1000))).to(torch.int32)
        top_p = 0.5 + 0.49 * rand(B)
        min_p = 0.2 * rand(B) ** 2
        kind = torch.randint(0, 6, (B,), device="cuda", generator=gen)
        if case["mix"] == "nucleus":
            top_k, min_p = torch.zeros_like(top_k), torch.zeros_like(min_p)
        elif case["mix"] == "topk":
            top_p, min_p = torch.ones_like(top_p), torch.zeros_like(min_p)
        else:
            top_k = torch.where((kind == 0) | (kind == 1), 0, top_k)
            top_p = torch.where((kind == 1) | (kind == 2), 1.0, top_p)
            min_p = torch.where((kind == 3) | (kind == 1), 0.0, min_p)
            temperature = torch.where(kind == 5, 0.0, temperature)
        return {"case": case, "logits": logits.to(t), "u": rand(B), "temperature": temperature,
                "top_k": top_k.to(torch.int32), "top_p": top_p, "min_p": min_p}
    hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
    n = case["rows"] if case["op"] == "step" else case["tokens"]
    silu = torch.nn.functional.silu
    # q, k and v as they leave a causal convolution and SiLU; keys that are not scaled here come at unit length
    q, k, v = (silu(randn(n, h, d, dtype=torch.float16).float()) for h, d in ((hk, dk), (hk, dk), (hv, dv)))
    if not case["norm"]:
        q, k = (x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS) for x in (q, k))
    dt = torch.exp(math.log(1e-3) + rand(hv) * (math.log(1e-1) - math.log(1e-3)))
    s = {"case": case, "q": q.to(t), "k": k.to(t), "v": v.to(t), "a": randn(n, hv).to(t), "b": randn(n, hv).to(t),
         "A_log": torch.log(1.0 + 15.0 * rand(hv)), "dt_bias": dt + torch.log(-torch.expm1(-dt)), "scale": dk ** -0.5}
    seqs = n if case["op"] == "step" else case["seqs"]
    slots = case.get("slots", seqs)
    s["state"] = 0.1 * randn(slots, hv, dv, dk)
    if case["op"] == "step":
        s["slots"] = torch.randperm(slots, device="cuda", generator=gen)[:n].to(torch.int32)
        return s
    lens = _lengths(case, seed)
    s["state"] *= (rand(seqs) < 0.5).float()[:, None, None, None]  # half of the sequences start anew
    s["slots"] = torch.randperm(seqs, device="cuda", generator=gen).to(torch.int32)
    starts = np.concatenate([[0], np.cumsum(lens)])
    s["lens"], s["cu_seqlens"] = lens, torch.tensor(starts, dtype=torch.int32, device="cuda")
    # the plain form's plan: the tokens of every chunk, and which chunks come c-th in their sequences
    rows = [(i, c) for i, length in enumerate(lens) for c in range(-(-length // CHUNK))]
    at = np.array([[starts[i] + c * CHUNK + j if c * CHUNK + j < lens[i] else n for j in range(CHUNK)] for i, c in rows],
                  dtype=np.int64).reshape(-1, CHUNK)
    s["tokens_of"] = torch.from_numpy(at).cuda()
    s["turns"] = []
    for c in range(-(-max(lens) // CHUNK)):
        now = [(j, i) for j, (i, cc) in enumerate(rows) if cc == c]
        s["turns"].append((torch.tensor([j for j, _ in now], device="cuda"), torch.tensor([i for _, i in now], device="cuda")))
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _unit(x, norm):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS) if norm else x


def _gates(s):
    """Log decay (64 bits: sums of it stand in exponents) and beta of every token and head."""
    x = s["a"].double() + s["dt_bias"].double()
    g = -torch.exp(s["A_log"].double()) * torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20.0))))
    return g, torch.sigmoid(s["b"].float())


def _step_plain(s):
    rep = s["case"]["hv"] // s["case"]["hk"]
    q, k = (_unit(s[x].float(), s["case"]["norm"]).repeat_interleave(rep, 1) for x in ("q", "k"))
    g, beta = _gates(s)
    at = s["slots"].long()
    S = s["state"][at] * torch.exp(g).float()[:, :, None, None]
    u = beta[:, :, None] * (s["v"].float() - (S * k[:, :, None, :]).sum(-1))
    S = S + u[:, :, :, None] * k[:, :, None, :]
    o = s["scale"] * (S * q[:, :, None, :]).sum(-1)
    s["state"][at] = S
    return {"o": o.to(s["v"].dtype), "state": s["state"]}


def _prefill_plain(s):
    """The chunked form: inside a chunk of 64 tokens the corrections u solve (I + L) u = beta (v - e^g S k) with L
    strictly lower triangular, so a chunk is a few matrix products and only the state goes from chunk to chunk."""
    case, at = s["case"], s["tokens_of"]
    rep = case["hv"] // case["hk"]
    n = s["q"].shape[0]

    def chunks(x):  # [tokens, heads, ...] -> [chunks, heads, 64, ...], zero past a sequence's end
        x = torch.cat([x, x.new_zeros(1, *x.shape[1:])])[at]
        return x.transpose(1, 2)

    q, k = (chunks(_unit(s[x].float(), case["norm"])).repeat_interleave(rep, 1) for x in ("q", "k"))
    v = chunks(s["v"].float())
    g, beta = _gates(s)
    g, beta = torch.cumsum(chunks(g), -1), chunks(beta)
    decay = g[..., :, None] - g[..., None, :]
    upto = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device="cuda").tril()
    decay = torch.exp(torch.where(upto, decay, 0.0)).float() * upto
    grow, last, left = torch.exp(g).float(), torch.exp(g[..., -1]).float(), torch.exp(g[..., -1:] - g).float()
    L = (beta[..., None] * (k @ k.transpose(-1, -2)) * decay).tril(-1)
    T = torch.eye(CHUNK, device="cuda").expand_as(L).clone()
    for i in range(1, CHUNK):  # forward substitution, every chunk at once
        T[..., i, :i] = -(L[..., i, None, :i] @ T[..., :i, :i])[..., 0, :]
    P = s["scale"] * (q @ k.transpose(-1, -2)) * decay
    out = torch.zeros_like(v)
    for now, seq in s["turns"]:  # the recurrence over chunks, every sequence at once
        slot = s["slots"][seq].long()
        S, kc, qc = s["state"][slot], k[now], q[now]
        u = T[now] @ (beta[now][..., None] * (v[now] - grow[now][..., None] * (kc @ S.transpose(-1, -2))))
        out[now] = s["scale"] * grow[now][..., None] * (qc @ S.transpose(-1, -2)) + P[now] @ u
        s["state"][slot] = last[now][..., None, None] * S + (left[now][..., None] * u).transpose(-1, -2) @ kc
    o = torch.zeros(n + 1, case["hv"], case["dv"], device="cuda", dtype=s["v"].dtype)
    o[at] = out.transpose(1, 2).to(o.dtype)
    return {"o": o[:n], "state": s["state"]}


def _sample_plain(s):
    """Tokens in order of falling logit, the lower index first among equal ones; weights and their sums in 64 bits."""
    greedy = ~(s["temperature"] > 0)
    x = s["logits"].float() / torch.where(greedy, 1.0, s["temperature"])[:, None]
    top_k = torch.where(greedy, 1, s["top_k"])
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp(x.double() - x[:, :1].double())
    rank = torch.arange(x.shape[1], device="cuda")
    kept = (x > -math.inf) & ((top_k <= 0)[:, None] | (rank < top_k[:, None]))
    w = torch.where(kept, w, 0.0)
    before = torch.cumsum(w, -1) - w
    nucleus = (s["top_p"] >= 1)[:, None] | (before <= s["top_p"].double()[:, None] * w.sum(-1, keepdim=True))
    kept &= nucleus & ((w >= s["min_p"].double()[:, None]) | (rank == 0))
    w = torch.where(kept, w, 0.0)
    inverse = torch.zeros_like(w).scatter_(1, order, w)  # back in the order of the vocabulary
    upto = torch.cumsum(inverse, -1)
    token = (upto <= s["u"].double()[:, None] * upto[:, -1:]).sum(-1)
    prob = torch.gather(inverse, 1, token[:, None])[:, 0] / upto[:, -1]
    return {"token": token.to(torch.int32), "kept": kept.sum(-1).to(torch.int32), "prob": prob.float()}


def run(state):
    s, case = state, state["case"]
    if own:
        from dfssm_b200 import ops
        if case["op"] == "sample":
            token, kept, prob = ops.sample_filtered(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                                    top_p=s["top_p"], min_p=s["min_p"])
            return {"token": token, "kept": kept, "prob": prob}
        if case["op"] == "step":
            o = ops.gated_delta_step(s["q"], s["k"], s["v"], s["a"], s["b"], s["A_log"], s["dt_bias"], s["state"],
                                     slots=s["slots"], scale=s["scale"], qk_norm=case["norm"])
        else:
            o = ops.gated_delta_prefill(s["q"], s["k"], s["v"], s["a"], s["b"], s["A_log"], s["dt_bias"], s["state"],
                                        s["cu_seqlens"], slots=s["slots"], scale=s["scale"], qk_norm=case["norm"])
        return {"o": o, "state": s["state"]}
    return {"step": _step_plain, "prefill": _prefill_plain, "sample": _sample_plain}[case["op"]](s)


# ------------------------------------------------------------------------------------------------ floors


def work(case):
    if case["op"] == "sample":
        B, V = case["rows"], case["vocab"]
        return {"bytes": B * V * (4 if case["type"] == "fp32" else 2) + 32 * B, "flops": 2 * B * V}
    hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
    n = case["rows"] if case["op"] == "step" else case["tokens"]
    seqs = n if case["op"] == "step" else case["seqs"]
    per_token = 2 * (2 * hk * dk + 2 * hv * dv + 2 * hv)
    # decay, S k, the correction and S q: 7 operations on each element of the state for every token
    return {"bytes": n * per_token + 2 * seqs * hv * dv * dk * 4, "flops": 7 * n * hv * dv * dk}


# ------------------------------------------------------------------------------------------------ 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _sample_exact(s)
    return _delta_exact(s)


def _delta_exact(s):
    """The recurrence as it is defined, token by token."""
    case = s["case"]
    rep = case["hv"] // case["hk"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    if case["norm"]:
        q, k = q / torch.sqrt((q ** 2).sum(-1, keepdim=True) + EPS), k / torch.sqrt((k ** 2).sum(-1, keepdim=True) + EPS)
    alpha = torch.exp(-torch.exp(s["A_log"].double()) * torch.logaddexp(s["a"].double() + s["dt_bias"].double(), q.new_zeros(())))
    beta = 1 / (1 + torch.exp(-s["b"].double()))
    lens = s.get("lens") or [1] * case["rows"]
    start = np.concatenate([[0], np.cumsum(lens)])[:-1]
    by_length = sorted(range(len(lens)), key=lambda i: -lens[i])  # the sequences still running are always the first ones
    slots = s["slots"].long()[torch.tensor(by_length, device="cuda")]
    first = torch.tensor([int(start[i]) for i in by_length], device="cuda")
    S, o = s["state"][slots].double(), torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    for t in range(max(lens)):
        m = sum(1 for i in by_length if lens[i] > t) if len(lens) > 1 else 1
        at = first[:m] + t
        kt, qt = k[at].repeat_interleave(rep, 1), q[at].repeat_interleave(rep, 1)
        St = S[:m]
        St *= alpha[at][:, :, None, None]
        u = beta[at][:, :, None] * (v[at] - (St @ kt[..., None])[..., 0])
        St += u[..., None] * kt[:, :, None, :]
        o[at] = case["dk"] ** -0.5 * (St @ qt[..., None])[..., 0]
    state = s["state"].double()
    state[slots] = S
    return {"o": o, "state": state}


def _sample_exact(s):
    tokens, counts, probs = [], [], []
    host = {x: s[x].float().cpu().numpy() for x in ("logits", "u", "temperature", "top_p", "min_p")}
    top_k = s["top_k"].cpu().numpy()
    for r in range(s["case"]["rows"]):
        temp, k = host["temperature"][r], int(top_k[r])
        if not temp > 0:
            temp, k = np.float32(1), 1
        x = (host["logits"][r] / temp).astype(np.float64)
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        if k > 0:
            order = order[:k]
        w = np.exp(x[order] - x[order[0]])
        n = len(order)
        if host["top_p"][r] < 1:
            n = int(np.searchsorted(np.cumsum(w), float(host["top_p"][r]) * w.sum(), side="right")) + 1
        keep = [i for i in range(min(n, len(order))) if i == 0 or w[i] >= float(host["min_p"][r])]
        index, weight = order[keep], w[keep]
        by = np.argsort(index)
        upto = np.cumsum(weight[by])
        j = int(np.searchsorted(upto, float(host["u"][r]) * upto[-1], side="right"))
        tokens.append(int(index[by][j]))
        counts.append(len(keep))
        probs.append(weight[by][j] / upto[-1])
    return {"token": np.array(tokens, np.int32), "kept": np.array(counts, np.int32), "prob": np.array(probs)}
