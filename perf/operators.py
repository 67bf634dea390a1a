"""Calls of the 8-bit integer products and of the log probabilities, with their sizes, inputs, work and
64-bit results: what a speed measurement of these operators runs.

Three operators:
  gemv     y = x W^T over int8 weights with a scale a channel (output row), the tokens' rows quantized to
           int8 with a scale a token inside the call
  gate_up  silu(gate x) * (up x) over such weights, gate rows stacked on up rows
  logprobs of each row of logits: the log probability and rank of a given token, the entropy, and the
           most probable tokens with their log probabilities

`run` computes them in their plain form (elementary torch operations), or, where `own` is true, through the
package's entry points.  Weights are N(0, 0.02) quantized a channel, held as rows on 128-byte lines, as a
program holds them after load.  Activations are N(0, 1) with a few channels eight times as large, as they
are behind a norm.  Logits are wide noise with a few likely tokens a row.
"""
import math

import torch

own = False

DT = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
SIZE = {"F32": 4, "F16": 2, "BF16": 2}


def listed():
    return [
        # one decoded token through a small square projection: a launch's latency
        {"name": "row_4096", "op": "gemv", "type": "BF16", "n": 4096, "k": 4096, "rows": 1, "bias": False},
        # the down-projection of a feed-forward block for a few sequences decoded together
        {"name": "down_6_rows", "op": "gemv", "type": "F32", "n": 4096, "k": 14336, "rows": 6, "bias": False},
        # the QKV projection with its bias for a batch of sequences decoded together
        {"name": "qkv_32_rows", "op": "gemv", "type": "BF16", "n": 6144, "k": 4096, "rows": 32, "bias": True},
        # a short prompt of odd length over a model with odd widths
        {"name": "odd_333_rows", "op": "gemv", "type": "F16", "n": 5003, "k": 2011, "rows": 333, "bias": False},
        # a long prompt through the feed-forward up-projection
        {"name": "prefill_2048", "op": "gemv", "type": "BF16", "n": 14336, "k": 4096, "rows": 2048, "bias": False},
        # the gate/up half of a feed-forward block, one decoded token
        {"name": "ffn_row", "op": "gate_up", "type": "BF16", "n": 14336, "k": 4096, "rows": 1},
        # the same of a narrower model over a short prompt of odd length, F32 as the other ops take it
        {"name": "ffn_200_rows", "op": "gate_up", "type": "F32", "n": 5632, "k": 2048, "rows": 200},
        # the same over a prompt
        {"name": "ffn_1024_rows", "op": "gate_up", "type": "BF16", "n": 14336, "k": 4096, "rows": 1024},
        # one decoded token's logits, no alternatives asked for: latency
        {"name": "token_1_row", "op": "logprobs", "type": "F32", "vocab": 32064, "rows": 1, "top": 0, "scale": 1.0,
         "hidden": 0.0},
        # a batch of decoded sequences, each with its alternatives, sampled at a temperature of 0.8
        {"name": "tokens_24_rows", "op": "logprobs", "type": "F32", "vocab": 128256, "rows": 24, "top": 20,
         "scale": 1.25, "hidden": 0.0},
        # a constrained batch: a grammar hides most of an odd vocabulary
        {"name": "masked_100_rows", "op": "logprobs", "type": "F16", "vocab": 50257, "rows": 100, "top": 5, "scale": 1.0,
         "hidden": 0.95},
        # every token of a long prompt scored against the next one
        {"name": "prompt_2048_rows", "op": "logprobs", "type": "BF16", "vocab": 128256, "rows": 2048, "top": 8,
         "scale": 1.0, "hidden": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same kinds: sizes from small models to large ones, odd ones among them, one token to
    a long prompt."""
    op, ty = rng.choice(["gemv", "gemv", "gate_up", "logprobs", "logprobs"]), rng.choice(["F32", "BF16", "BF16", "F16"])
    if op == "logprobs":
        top = rng.choice([0, 1, 5, 20, rng.randint(1, 64)])
        return {"op": op, "type": ty, "vocab": _log(rng, 1000, 128256), "rows": _log(rng, 1, 1024), "top": top,
                "scale": rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)]), "hidden": rng.choice([0.0, 0.0, 0.9])}
    unit = rng.choice([1, 16, 128, 128])
    k = unit * _log(rng, -(-512 // unit), (14336 if op == "gemv" else 4096) // unit)
    n = _log(rng, 512, 14336)
    rows = _log(rng, 1, 2048 if k <= 4096 and op == "gemv" else 512)
    c = {"op": op, "type": ty, "n": n, "k": k, "rows": rows}
    if op == "gemv":
        c["bias"] = rng.random() < 0.3
    return c


# ---- inputs ---------------------------------------------------------------------------------------

def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * (int(seed) % (1 << 40)) + part)
    return g


def _normal(seed, part, *shape):
    return torch.randn(*shape, generator=_gen(seed, part), device="cuda", dtype=torch.float32)


def _logits(c, seed):
    rows, vocab = c["rows"], c["vocab"]
    x = 2.0 * _normal(seed, 1, rows, vocab)
    likely = torch.randint(vocab, (rows, 8), generator=_gen(seed, 2), device="cuda")
    x.scatter_(1, likely, 9.0 + 2.0 * _normal(seed, 3, rows, 8))
    other = torch.randint(vocab, (rows,), generator=_gen(seed, 4), device="cuda")
    pick = torch.rand(rows, generator=_gen(seed, 5), device="cuda") < 0.7
    token = torch.where(pick, likely[:, 0], other)
    if c["hidden"]:
        hide = torch.rand(rows, vocab, generator=_gen(seed, 6), device="cuda") < c["hidden"]
        hide.scatter_(1, token.unsqueeze(1), False)
        x.masked_fill_(hide, float("-inf"))
    if rows > 1:
        token[-1] = -1  # the last row has no next token
    return x.to(DT[c["type"]]), token


def _weights(c, seed):
    n, k = (2 if c["op"] == "gate_up" else 1) * c["n"], c["k"]
    w = 0.02 * _normal(seed, 1, n, k)
    scales = w.abs().amax(1) / 127.0
    codes = torch.zeros(n, -(-k // 128) * 128, dtype=torch.int8, device="cuda")[:, :k]
    codes.copy_(torch.round(w / scales.unsqueeze(1)).clamp_(-127, 127))
    bias = _normal(seed, 2, n) if c.get("bias") else None
    x = _normal(seed, 3, c["rows"], k)
    x *= 1.0 + 7.0 * (torch.rand(k, generator=_gen(seed, 4), device="cuda") < 0.01)
    return codes, scales, bias, x.to(DT[c["type"]])


def prepare(case, seed):
    c = case
    if c["op"] == "logprobs":
        x, token = _logits(c, seed)
        return {"c": c, "x": x, "token": token}
    codes, scales, bias, x = _weights(c, seed)
    st = {"c": c, "codes": codes, "scales": scales, "bias": bias, "x": x}
    if own:  # the handle on these tensors that a program keeps
        import syntropy_amd.int8 as I
        st["w"] = I.Weights(codes, scales, bias)
    return st


# ---- the plain forms --------------------------------------------------------------------------------

def _product(codes, scales, bias, x):
    """The product in F32: the tokens' codes and scales, the sum, both scales, the bias."""
    x = x.to(torch.float32)
    s = x.abs().amax(1, keepdim=True) / 127.0
    inv = 1.0 / s
    q = torch.round(x * torch.where(torch.isfinite(inv), inv, 0.0))
    y = torch.matmul(q, codes.to(torch.float32).t()) * s * scales
    return y if bias is None else y + bias


def _plain_logprobs(c, x, token):
    v = x.to(torch.float32)
    z = v * c["scale"]
    m = z.amax(1, keepdim=True)
    seen = m > -math.inf
    d = torch.where(seen, z - m, -math.inf)
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    lse = torch.log(s)
    entropy = torch.where(seen, lse - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / s, 0.0).squeeze(1)
    at = token.clamp(min=0).unsqueeze(1)
    logprob = torch.where(token < 0, 0.0, torch.where(seen, d.gather(1, at) - lse, -math.inf).squeeze(1))
    rank = torch.where(token < 0, -1, (v > v.gather(1, at)).sum(1)).to(torch.int32)
    if c["top"]:
        # a whole number that orders as (value descending, index ascending)
        b = (v + 0.0).view(torch.int32)
        b = torch.where(b < 0, b ^ 0x7FFFFFFF, b).to(torch.int64)
        key = (b << 32) | (0xFFFFFFFF - torch.arange(c["vocab"], device=x.device))
        ids = 0xFFFFFFFF - (torch.topk(key, c["top"], 1).values & 0xFFFFFFFF)
    else:
        ids = torch.empty(c["rows"], 0, dtype=torch.int64, device=x.device)
    top = torch.where(seen, d.gather(1, ids) - lse, -math.inf)
    return logprob, rank, entropy, ids.to(torch.int32), top


def run(state):
    c = state["c"]
    if own:
        if c["op"] == "logprobs":
            import syntropy_amd.gemv as S
            r = S.token_logprobs(state["x"], state["token"], top=c["top"], scale=c["scale"])
            return r.logprob, r.rank, r.entropy, r.top_ids, r.top_logprobs
        import syntropy_amd.int8 as I
        return (I.gate_up_act if c["op"] == "gate_up" else I.gemv)(state["w"], state["x"], c["rows"])
    if c["op"] == "logprobs":
        return _plain_logprobs(c, state["x"], state["token"])
    y = _product(state["codes"], state["scales"], state["bias"], state["x"])
    if c["op"] == "gate_up":
        g, u = y[:, :c["n"]], y[:, c["n"]:]
        y = g / (1.0 + torch.exp(-g)) * u
    return y.to(DT[c["type"]])


def work(case):
    c = case
    es, rows = SIZE[c["type"]], c["rows"]
    if c["op"] == "logprobs":
        # a value is scaled, compared, shifted, exponentiated, and added to two sums
        return {"bytes": rows * (c["vocab"] * es + 8 + 12 + 8 * c["top"]), "flops": 7 * rows * c["vocab"]}
    n = (2 if c["op"] == "gate_up" else 1) * c["n"]
    return {"bytes": n * c["k"] + (8 if c.get("bias") else 4) * n + es * rows * (c["k"] + c["n"]),
            "flops": 2 * n * c["k"] * rows}


# ---- the same in 64 bits ----------------------------------------------------------------------------

def _exact_logprobs(c, seed):
    x, token = _logits(c, seed)
    lp, rank, ent, ids, tlp = [], [], [], [], []
    for r in range(c["rows"]):
        v = x[r].to(torch.float64)
        z = v * c["scale"]
        lse = torch.logsumexp(z, 0)
        logp = z - lse
        p = torch.exp(logp)
        ent.append(-torch.where(p > 0, p * logp, torch.zeros_like(p)).sum())
        t = token[r]
        lp.append(torch.where(t < 0, torch.zeros_like(lse), logp[t]))
        rank.append(torch.where(t < 0, torch.full_like(t, -1), (v > v[t]).sum()))
        first = torch.sort(v, descending=True, stable=True).indices[:c["top"]]
        ids.append(first)
        tlp.append(logp[first])
    return (torch.stack(lp), torch.stack(rank).to(torch.int32), torch.stack(ent), torch.stack(ids).to(torch.int32),
            torch.stack(tlp))


def exact(case, seed):
    c = case
    if c["op"] == "logprobs":
        return _exact_logprobs(c, seed)
    codes, scales, bias, x = _weights(c, seed)
    # a token's scale, its inverse and its codes are defined by F32 steps; all that follows is real numbers
    d = torch.linalg.vector_norm(x.to(torch.float32), float("inf"), 1, keepdim=True) / torch.full((), 127.0, device="cuda")
    q = (x.to(torch.float32) * torch.reciprocal(d.to(torch.float64)).to(torch.float32)).round().to(torch.float64)
    y = (q @ codes.to(torch.float64).T) * (d.to(torch.float64) * scales.to(torch.float64))
    if bias is not None:
        y = y + bias.to(torch.float64)
    if c["op"] == "gate_up":
        y = torch.nn.functional.silu(y[:, :c["n"]]) * y[:, c["n"]:]
    return y
