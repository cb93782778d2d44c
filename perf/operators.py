"""Cases of the operators at the two vocabulary ends of a language model's training step.

Three operators: the cross-entropy of a linear head whose logits are never handed out (``linear_cross_entropy``),
the distillation of such a head from a teacher's top logits (``linear_distillation``) and the scaled embedding
lookup whose weight gradient is summed over tokens sorted by id (``scaled_embedding``).

``own`` selects the side: False runs each operator in its plain form (elementary torch operations in 32 bits,
rounded once at the end), True runs the framework's operators.
"""
from __future__ import annotations

import math

import torch

own = False


# ------------------------------------------------------------------------------------------------ cases
def _head(name, T, H, V, mode, ignored):
    return {"name": name, "op": "linear_cross_entropy", "T": T, "H": H, "V": V, "mode": mode, "ignored": ignored}


def _distill(name, T, H, V, K, temperature, values, ignored):
    return {"name": name, "op": "linear_distillation", "T": T, "H": H, "V": V, "K": K, "temperature": temperature,
            "values": values, "ignored": ignored}


def _embed(name, T, H, V, dtype, scale, shard):
    return {"name": name, "op": "scaled_embedding", "T": T, "H": H, "V": V, "dtype": dtype, "scale": scale,
            "shard": shard}


def listed():
    return [
        # a toy model's step: the call's own latency counts
        _head("ce_toy_t64_h256_v1000", 64, 256, 1000, "mean", 0.1),
        # the default GPT-2 block's head: one 2048-token sequence shifted by one, odd vocabulary
        _head("ce_gpt2_t2047_h768_v50257", 2047, 768, 50257, "mean", 0.0),
        # GPT-1.3B shape: a micro-batch of 8 sequences of 2048 tokens
        _head("ce_gpt13b_t16384_h2048_v50304", 16384, 2048, 50304, "mean", 0.02),
        # Llama-8B shape: two sequences of 4096 tokens, the prompt's tokens masked out
        _head("ce_llama8b_t8192_h4096_v128256", 8192, 4096, 128256, "mean", 0.25),
        # one loss for each token, weighted by the caller (a policy's advantages): per-row upstream gradients
        _head("ce_rows_t1500_h2048_v102400", 1500, 2048, 102400, "rows", 0.1),
        # scoring a short continuation: the log-probabilities alone, no gradient
        _head("ce_score_t17_h4096_v128256", 17, 4096, 128256, "score", 0.0),
        # a toy student
        _distill("kd_toy_t96_h512_v1024_k8", 96, 512, 1024, 8, 1.0, "float32", 0.1),
        # DeepSeek-V2-Lite-shape student, softened targets kept in 16 bits
        _distill("kd_dsv2lite_t4096_h2048_v102400_k64", 4096, 2048, 102400, 64, 2.0, "bfloat16", 0.1),
        # Llama-8B-shape student, an odd number of teacher logits
        _distill("kd_llama8b_t4000_h4096_v128256_k101", 4000, 4096, 128256, 101, 1.0, "float32", 0.2),
        # a toy model's lookup
        _embed("emb_toy_t64_h256_v1000", 64, 256, 1000, "bfloat16", 1.0, 0),
        # the default GPT-2 block in fp32
        _embed("emb_gpt2_t8192_h768_v50257_fp32", 8192, 768, 50257, "float32", 1.0, 0),
        # Llama-8B shape: 8 sequences of 4096 tokens, outputs scaled by sqrt(H)
        _embed("emb_llama8b_t32768_h4096_v128256", 32768, 4096, 128256, "bfloat16", 64.0, 0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear_cross_entropy", "linear_cross_entropy", "linear_distillation", "scaled_embedding"])
    H = 8 * _log_int(rng, 8, 512)
    if H == 3072:
        H += 8
    V = _log_int(rng, 300, 128256)
    if op == "scaled_embedding":
        T = _log_int(rng, 1, 32768)
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        if dtype == "float32":
            H = min(H, 2048)
        H -= rng.choice([0, 0, 0, 1, 4])  # rows that are no multiple of 16 bytes
        return _embed(None, T, H, V, dtype, rng.choice([1.0, math.sqrt(H), 0.5]), rng.choice([0, 0, 1]))
    T = _log_int(rng, 1, 8192)
    ignored = rng.choice([0.0, 0.1, 0.5])
    if op == "linear_cross_entropy":
        return _head(None, T, H, V, rng.choice(["mean", "mean", "rows", "score"]), ignored)
    K = min(_log_int(rng, 1, 256), int(math.sqrt(V / 4)))
    return _distill(None, min(T, 4096), H, V, max(1, K), rng.choice([1.0, 1.0, 2.0, 0.7]),
                    rng.choice(["float32", "bfloat16"]), ignored)


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)


def _frequent(g, n, V):
    """Token ids with a 1/(rank + 3) frequency, as text has: a few ids are in many tokens, most in none."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    return (3.0 * torch.exp(u * math.log((V + 3.0) / 3.0)) - 3.0).long().clamp_(0, V - 1)


def _head_inputs(g, T, H, V, near):
    """Final hidden states (unit RMS, leaning towards the row that is to be predicted) and the head's weight."""
    w = torch.empty(V, H, device="cuda", dtype=torch.bfloat16).normal_(0.0, 0.02, generator=g)
    h = torch.randn(T, H, device="cuda", generator=g)
    lean = torch.rand(T, 1, device="cuda", generator=g) * (12.0 / 0.02 / math.sqrt(H))
    h = h + lean * w[near].float()
    h = h * torch.rsqrt(h.square().mean(-1, keepdim=True))
    return h.to(torch.bfloat16).requires_grad_(True), w.requires_grad_(True)


def prepare(case, seed):
    g = _generator(seed)
    T, H, V, op = case["T"], case["H"], case["V"], case["op"]
    if op == "scaled_embedding":
        dtype = getattr(torch, case["dtype"])
        start = V if case["shard"] else 0  # the second of two shards of a vocabulary of 2 V
        ids = _frequent(g, T, 2 * V if case["shard"] else V)
        w = torch.empty(V, H, device="cuda", dtype=dtype).normal_(0.0, 0.02, generator=g).requires_grad_(True)
        dout = (torch.randn(T, H, device="cuda", generator=g) * 1e-3).to(dtype)
        return {"op": op, "ids": ids, "w": w, "dout": dout, "scale": case["scale"], "start": start}
    if op == "linear_cross_entropy":
        labels = _frequent(g, T, V)
        h, w = _head_inputs(g, T, H, V, labels)
        labels = torch.where(torch.rand(T, device="cuda", generator=g) < case["ignored"], -100, labels)
        rows = torch.randn(T, device="cuda", generator=g) / T
        return {"op": op, "mode": case["mode"], "h": h, "w": w, "labels": labels, "rows": rows}
    # One teacher id from each of K ranges of the vocabulary, the low (frequent) ids in the narrow ranges.
    K = case["K"]
    edge = torch.tensor([int(V * (k / K) ** 2) for k in range(K + 1)], device="cuda")
    u = torch.rand(T, K, device="cuda", generator=g)
    idx = edge[:-1] + (u * (edge[1:] - edge[:-1])).long().clamp_min(0)
    idx = torch.minimum(idx, edge[1:] - 1)
    order = torch.rand(T, K, device="cuda", generator=g).argsort(1)
    idx = idx.gather(1, order)
    gaps = -torch.log(torch.rand(T, K, device="cuda", generator=g).clamp_min(1e-6)) * 0.5
    values = (15.0 + torch.randn(T, 1, device="cuda", generator=g) - gaps.cumsum(1).clamp_max(25.0))
    values = values.to(getattr(torch, case["values"]))
    h, w = _head_inputs(g, T, H, V, idx[:, 0])
    idx = torch.where(torch.rand(T, 1, device="cuda", generator=g) < case["ignored"], -1, idx)
    return {"op": op, "h": h, "w": w, "values": values, "indices": idx, "temperature": case["temperature"]}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


def _run_own(s):
    from nano_train_b200 import ops

    if s["op"] == "scaled_embedding":
        out = ops.scaled_embedding(s["ids"], s["w"], s["scale"], vocab_start=s["start"])
        (dw,) = torch.autograd.grad(out, (s["w"],), s["dout"])
        return {"out": out.detach(), "dw": dw}
    if s["op"] == "linear_cross_entropy":
        if s["mode"] == "score":
            with torch.no_grad():
                return {"loss": ops.linear_cross_entropy(s["h"], s["w"], s["labels"], reduction="none")}
        if s["mode"] == "rows":
            loss = ops.linear_cross_entropy(s["h"], s["w"], s["labels"], reduction="none")
            dh, dw = torch.autograd.grad(loss, (s["h"], s["w"]), s["rows"])
        else:
            loss = ops.linear_cross_entropy(s["h"], s["w"], s["labels"])
            dh, dw = torch.autograd.grad(loss, (s["h"], s["w"]))
        return {"loss": loss.detach(), "dh": dh, "dw": dw}
    loss = ops.linear_distillation(s["h"], s["w"], s["values"], s["indices"], temperature=s["temperature"])
    dh, dw = torch.autograd.grad(loss, (s["h"], s["w"]))
    return {"loss": loss.detach(), "dh": dh, "dw": dw}


def _run_plain(s):
    if s["op"] == "scaled_embedding":
        w, local = s["w"], s["ids"] - s["start"]
        inside = (local >= 0) & (local < w.shape[0])
        local = torch.where(inside, local, 0)
        keep = inside[:, None].float() * s["scale"]
        out = (w[local].float() * keep).to(w.dtype)
        dw = torch.zeros(w.shape, device=w.device).index_add_(0, local, s["dout"].float() * keep).to(w.dtype)
        return {"out": out, "dw": dw}
    h, w = s["h"], s["w"]
    hf, wf = h.float(), w.float()
    logits = hf @ wf.t()
    if s["op"] == "linear_cross_entropy":
        valid = s["labels"] >= 0
        target = torch.where(valid, s["labels"], 0)[:, None]
        top = logits.max(1, keepdim=True).values
        lse = top + (logits - top).exp().sum(1, keepdim=True).log()
        rows = torch.where(valid, (lse - logits.gather(1, target))[:, 0], 0.0)
        if s["mode"] == "score":
            return {"loss": rows}
        count = valid.sum().clamp_min(1)
        scale = s["rows"] if s["mode"] == "rows" else torch.ones_like(rows) / count
        g = (logits - lse).exp()
        g.scatter_add_(1, target, torch.full_like(lse, -1.0))
        g *= (scale * valid)[:, None]
        loss = rows if s["mode"] == "rows" else rows.sum() / count
        return {"loss": loss, "dh": (g @ wf).to(h.dtype), "dw": (g.t() @ hf).to(w.dtype)}
    tau = s["temperature"]
    present = s["indices"] >= 0
    valid = present.any(1)
    idx = torch.where(present, s["indices"], 0)
    v = torch.where(present, s["values"].float() / tau, -math.inf)
    v = v - torch.where(valid[:, None], v.max(1, keepdim=True).values, 0.0)
    e = v.exp()
    q = e / torch.where(valid[:, None], e.sum(1, keepdim=True), 1.0)
    logits /= tau
    top = logits.max(1, keepdim=True).values
    lse = top + (logits - top).exp().sum(1, keepdim=True).log()
    logq = torch.where(q > 0, q, 1.0).log()
    rows = (q * (logq - (logits.gather(1, idx) - lse))).sum(1)
    count = valid.sum().clamp_min(1)
    g = (logits - lse).exp()
    g.scatter_add_(1, idx, -q)
    g *= (valid * (tau / count))[:, None]
    return {"loss": rows.sum() * (tau * tau) / count, "dh": (g @ wf).to(h.dtype), "dw": (g.t() @ hf).to(w.dtype)}


# ------------------------------------------------------------------------------------------------ floors
def _distinct(T, V):
    """Expected number of distinct ids among T draws of ``_frequent``."""
    v = torch.arange(V, dtype=torch.float64)
    p = torch.log((v + 4.0) / (v + 3.0)) / math.log((V + 3.0) / 3.0)
    return float((1.0 - (1.0 - p).pow(T)).sum())


def work(case):
    T, H, V, op = case["T"], case["H"], case["V"], case["op"]
    if op == "scaled_embedding":
        size = 2 if case["dtype"] == "bfloat16" else 4
        rows = _distinct(T, 2 * V) / 2 if case["shard"] else _distinct(T, V)
        # ids, the rows looked up and the upstream gradient in; the lookup and the weight gradient out
        return {"bytes": 8 * T + size * H * (rows + 2 * T + V), "flops": 2 * T * H}
    ends = 2 * H * (T + V)
    if op == "linear_cross_entropy":
        if case["mode"] == "score":
            return {"bytes": ends + 12 * T, "flops": 2 * T * V * H}
        extra = 16 * T if case["mode"] == "rows" else 8 * T + 4
        return {"bytes": 2 * ends + extra, "flops": 6 * T * V * H}
    size = 2 if case["values"] == "bfloat16" else 4
    return {"bytes": 2 * ends + T * case["K"] * (8 + size) + 4, "flops": 6 * T * V * H}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The operators from their definitions in 64 bits, a slice of the tokens at a time."""
    s = prepare(case, seed)
    with torch.no_grad():
        if s["op"] == "scaled_embedding":
            table = torch.cat([s["w"].double(), s["w"].new_zeros(1, case["H"], dtype=torch.float64)])
            V = case["V"]
            row = s["ids"] - s["start"]
            row[(row < 0) | (row >= V)] = V  # the added row of zeros
            grad = torch.zeros_like(table)
            grad.index_put_((row,), s["dout"].double() * s["scale"], accumulate=True)
            return {"out": table[row] * s["scale"], "dw": grad[:V]}
        h, w = s["h"].double(), s["w"].double()
        tau = s.get("temperature", 1.0)
        T = h.shape[0]
        dh, dw, rows = torch.zeros_like(h), torch.zeros_like(w), h.new_zeros(T)
        if s["op"] == "linear_cross_entropy":
            keep = s["labels"] != -100
            upstream = s["rows"].double() if s["mode"] == "rows" else h.new_full((T,), 1.0 / max(1, int(keep.sum())))
        else:
            keep = (s["indices"] >= 0).any(1)
            upstream = h.new_full((T,), 1.0 / max(1, int(keep.sum())))
        for a in range(0, T, 1024):
            b = min(T, a + 1024)
            live = keep[a:b].nonzero()[:, 0] + a
            if live.numel() == 0:
                continue
            logp = torch.log_softmax(h[live] @ w.t() / tau, 1)
            wanted = torch.zeros_like(logp)
            if s["op"] == "linear_cross_entropy":
                pick = s["labels"][live][:, None]
                wanted.scatter_(1, pick, 1.0)
                rows[live] = -logp.gather(1, pick)[:, 0]
            else:
                there = s["indices"][live] >= 0
                pick = s["indices"][live].clamp_min(0)
                score = (s["values"][live].double() / tau).masked_fill(~there, -math.inf)
                logq = torch.log_softmax(score, 1)
                q = logq.exp()
                wanted.scatter_add_(1, pick, q)
                terms = q * (logq.masked_fill(~there, 0.0) - logp.gather(1, pick))
                rows[live] = tau * tau * terms.sum(1)
            if s.get("mode") == "score":
                continue
            g = (logp.exp_() - wanted) * (tau * upstream[live])[:, None]
            dh[live] = g @ w
            dw += g.t() @ h[live]
        if s.get("mode") == "score":
            return {"loss": rows}
        loss = rows if s.get("mode") == "rows" else (rows * upstream).sum()
        return {"loss": loss, "dh": dh, "dw": dw}
