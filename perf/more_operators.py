"""Calls of what stands around a model's products in a step, with their sizes, inputs, work and 64-bit
results: what a speed measurement of these operators runs.

Three operators:
  product  y = act(x W^T + bias) * gate + residual over F16 or BF16 weights and activations; bias, activation,
           gate and residual each there or not
  norm     the end of one block and the beginning of the next: h = x + scale * gate * a, where a is the block's
           output or its RmsNorm, and y = RmsNorm(h)
  sample   a token of each row of logits by temperature, top-k, top-p and min-p from a given random number, its
           log probability among the tokens that were kept, and how many those are

`run` computes them in their plain form (elementary torch operations), or, where `own` is true, through the
package's entry points.  Weights are N(0, 0.02).  Activations are N(0, 1) with a few channels eight times as
large, as they are behind a norm; a residual stream is N(0, 4), a block's output N(0, 1).  Logits are wide noise
with a few likely tokens a row.
"""
import math

import torch

own = False

DT = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
SIZE = {"F32": 4, "F16": 2, "BF16": 2}
EPS = 1e-5


def listed():
    return [
        # one decoded token through the attention's output projection, added to the residual stream: latency
        {"name": "out_1_row", "op": "product", "type": "BF16", "out": "BF16", "n": 4096, "k": 4096, "rows": 1,
         "bias": False, "act": "none", "gate": False, "residual": True},
        # the down-projection of a feed-forward block for a few sequences decoded together, onto an F32 residual
        {"name": "down_6_rows", "op": "product", "type": "BF16", "out": "F32", "n": 4096, "k": 14336, "rows": 6,
         "bias": False, "act": "none", "gate": False, "residual": True},
        # the QKV projection with its bias for a batch of sequences decoded together
        {"name": "qkv_32_rows", "op": "product", "type": "F16", "out": "F16", "n": 6144, "k": 4096, "rows": 32,
         "bias": True, "act": "none", "gate": False, "residual": False},
        # a feed-forward block's first half over a short prompt of odd length, a model with odd widths
        {"name": "odd_333_rows", "op": "product", "type": "F16", "out": "F16", "n": 5003, "k": 2011, "rows": 333,
         "bias": True, "act": "gelu", "gate": False, "residual": False},
        # the gate projection of a gated feed-forward block over a long prompt, the up-projection's rows at hand
        {"name": "gated_2048_rows", "op": "product", "type": "BF16", "out": "BF16", "n": 14336, "k": 4096, "rows": 2048,
         "bias": False, "act": "silu", "gate": True, "residual": False},
        # between two blocks, one decoded token: latency
        {"name": "norm_1_row", "op": "norm", "type": "BF16", "stream": "BF16", "n": 4096, "rows": 1, "post": False,
         "gate": "none", "scale": 1.0},
        # a norm behind the block too, a gate a channel, an F32 stream, odd width and length
        {"name": "norm_333_rows", "op": "norm", "type": "F16", "stream": "F32", "n": 2011, "rows": 333, "post": True,
         "gate": "channel", "scale": 0.5},
        # the same with a gate a token and channel over a long prompt
        {"name": "norm_8192_rows", "op": "norm", "type": "BF16", "stream": "BF16", "n": 4096, "rows": 8192, "post": True,
         "gate": "token", "scale": 0.22},
        # one sequence's next token by the usual filters: latency
        {"name": "token_1_row", "op": "sample", "type": "F32", "vocab": 32064, "rows": 1, "temperature": 0.8, "top_k": 40,
         "top_p": 0.95, "min_p": 0.0, "each": False, "hidden": 0.0},
        # a batch of sequences, a wide vocabulary, the nucleus alone
        {"name": "nucleus_24_rows", "op": "sample", "type": "F32", "vocab": 128256, "rows": 24, "temperature": 1.0,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0, "each": False, "hidden": 0.0},
        # a constrained batch: a grammar hides most of an odd vocabulary
        {"name": "masked_100_rows", "op": "sample", "type": "F16", "vocab": 50257, "rows": 100, "temperature": 1.25,
         "top_k": 0, "top_p": 1.0, "min_p": 0.02, "each": False, "hidden": 0.95},
        # a full server's batch, every sequence with its own settings
        {"name": "server_256_rows", "op": "sample", "type": "BF16", "vocab": 128256, "rows": 256, "temperature": 1.0,
         "top_k": 0, "top_p": 1.0, "min_p": 0.0, "each": True, "hidden": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same kinds: sizes from small models to large ones, odd ones among them, one token to
    a long prompt."""
    op = rng.choice(["product", "product", "product", "norm", "sample", "sample"])
    if op == "norm":
        n = rng.choice([1, 8, 128, 128])
        n *= _log(rng, -(-256 // n), 16384 // n)
        ty = rng.choice(["F32", "BF16", "BF16", "F16"])
        return {"op": op, "type": ty, "stream": rng.choice([ty, ty, "F32"]), "n": n, "rows": _log(rng, 1, min(8192, (1 << 25) // n)),
                "post": rng.random() < 0.5, "gate": rng.choice(["none", "channel", "token"]),
                "scale": rng.choice([1.0, round(rng.uniform(0.1, 2.0), 3)])}
    if op == "sample":
        return {"op": op, "type": rng.choice(["F32", "F32", "BF16", "F16"]), "vocab": _log(rng, 1000, 128256),
                "rows": _log(rng, 1, 256), "temperature": round(rng.uniform(0.5, 1.5), 3),
                "top_k": rng.choice([0, 0, 1, 20, 50, rng.randint(2, 500)]),
                "top_p": rng.choice([1.0, 0.95, 0.9, round(rng.uniform(0.3, 0.999), 3)]),
                "min_p": rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0.001, 0.2), 3)]), "each": rng.random() < 0.25,
                "hidden": rng.choice([0.0, 0.0, 0.0, 0.9])}
    unit = rng.choice([1, 8, 128, 128])
    ty = rng.choice(["BF16", "BF16", "F16"])
    k = unit * _log(rng, -(-512 // unit), 14336 // unit)
    n = rng.choice([1, 8])
    n *= _log(rng, -(-512 // n), 14336 // n)
    return {"op": op, "type": ty, "out": rng.choice([ty, ty, "F32"]), "n": n, "k": k,
            "rows": _log(rng, 1, 2048 if n * k <= 14336 * 4096 else 512), "bias": rng.random() < 0.3,
            "act": rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh"]), "gate": rng.random() < 0.25,
            "residual": rng.random() < 0.5}


# ---- inputs ---------------------------------------------------------------------------------------

def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * (int(seed) % (1 << 40)) + part)
    return g


def _normal(seed, part, *shape):
    return torch.randn(*shape, generator=_gen(seed, part), device="cuda", dtype=torch.float32)


def _uniform(seed, part, *shape):
    return torch.rand(*shape, generator=_gen(seed, part), device="cuda", dtype=torch.float32)


def _product_inputs(c, seed):
    n, k, rows, ty, out = c["n"], c["k"], c["rows"], DT[c["type"]], DT[c["out"]]
    x = _normal(seed, 2, rows, k)
    x *= 1.0 + 7.0 * (_uniform(seed, 3, k) < 0.01)
    return {"w": (0.02 * _normal(seed, 1, n, k)).to(ty), "x": x.to(ty),
            "bias": 0.5 * _normal(seed, 4, n) if c["bias"] else None,
            "gate": _normal(seed, 5, rows, n).to(ty) if c["gate"] else None,
            "residual": (2.0 * _normal(seed, 6, rows, n)).to(out) if c["residual"] else None}


def _norm_inputs(c, seed):
    n, rows, ty = c["n"], c["rows"], DT[c["type"]]
    gate = None
    if c["gate"] != "none":
        gate = (1.0 + 0.5 * _normal(seed, 3, *((n,) if c["gate"] == "channel" else (rows, n)))).to(ty)
    return {"x": (2.0 * _normal(seed, 1, rows, n)).to(DT[c["stream"]]), "branch": _normal(seed, 2, rows, n).to(ty),
            "gate": gate, "post": 1.0 + 0.2 * _normal(seed, 4, n) if c["post"] else None,
            "g": 1.0 + 0.2 * _normal(seed, 5, n)}


def _sample_inputs(c, seed):
    rows, vocab = c["rows"], c["vocab"]
    x = 2.0 * _normal(seed, 1, rows, vocab)
    likely = torch.randint(vocab, (rows, 8), generator=_gen(seed, 2), device="cuda")
    # half of the rows are sure of a few tokens, half are not
    sure = torch.where(_uniform(seed, 9, rows, 1) < 0.5, 16.0, 9.0)
    x.scatter_(1, likely, sure + 2.0 * _normal(seed, 3, rows, 8))
    if c["hidden"]:
        hide = _uniform(seed, 6, rows, vocab) < c["hidden"]
        hide.scatter_(1, likely, False)
        x.masked_fill_(hide, float("-inf"))
    if not c["each"]:
        how = {key: c[key] for key in ("temperature", "top_k", "top_p", "min_p")}
    else:  # a few kinds of callers, some of them greedy
        r = [_uniform(seed, 20 + i, rows) for i in range(5)]
        how = {"temperature": torch.where(r[0] < 0.1, 0.0, 0.5 + r[1]),
               "top_k": torch.where(r[2] < 0.5, 0, (1 + 100 * r[3]).to(torch.int32)).to(torch.int32),
               "top_p": torch.where(r[4] < 0.3, 1.0, 0.5 + 0.49 * r[3]),
               "min_p": torch.where(r[4] > 0.7, 0.1 * r[1], 0.0)}
    return {"x": x.to(DT[c["type"]]), "u": _uniform(seed, 5, rows), "how": how}


INPUTS = {"product": _product_inputs, "norm": _norm_inputs, "sample": _sample_inputs}


def prepare(case, seed):
    st = {"c": case, **INPUTS[case["op"]](case, seed)}
    if own and case["op"] == "product":  # the handle on the matrix that a program keeps
        import syntropy_amd.half as H
        st["w"] = H.Weights(st["w"], st["bias"])
    return st


# ---- the plain forms --------------------------------------------------------------------------------

def _plain_product(c, st):
    v = torch.matmul(st["x"].to(torch.float32), st["w"].to(torch.float32).t())
    if c["bias"]:
        v = v + st["bias"]
    if c["act"] == "relu":
        v = torch.where(v > 0.0, v, 0.0)
    elif c["act"] == "silu":
        v = v / (1.0 + torch.exp(-v))
    elif c["act"] == "gelu":
        v = 0.5 * v * torch.special.erfc(v * -math.sqrt(0.5))
    elif c["act"] == "gelu_tanh":
        v = v / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if c["gate"]:
        v = v * st["gate"].to(torch.float32)
    if c["residual"]:
        v = v + st["residual"].to(torch.float32)
    return v.to(DT[c["out"]])


def _rms(v, g):
    return v * (1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)) * g


def _plain_norm(c, st):
    a = st["branch"].to(torch.float32)
    if c["post"]:
        a = _rms(a, st["post"])
    if c["gate"] != "none":
        a = a * st["gate"].to(torch.float32)
    h = st["x"].to(torch.float32) + c["scale"] * a
    return h.to(DT[c["stream"]]), _rms(h, st["g"]).to(DT[c["type"]])


def _plain_sample(c, st):
    """In 64 bits: a token and a count are whole numbers, and stand next to borders."""
    x, u = st["x"].to(torch.float32), st["u"].to(torch.float64)
    rows, vocab = x.shape
    t, k, p, mp = (v if torch.is_tensor(v) else torch.full((rows,), v, device=x.device)
                   for v in (st["how"][key] for key in ("temperature", "top_k", "top_p", "min_p")))
    # a whole number that orders as (value descending, index ascending)
    b = (x + 0.0).view(torch.int32)
    b = torch.where(b < 0, b ^ 0x7FFFFFFF, b).to(torch.int64)
    key = (b << 32) | (0xFFFFFFFF - torch.arange(vocab, device=x.device))
    ids = 0xFFFFFFFF - (torch.sort(key, 1, descending=True).values & 0xFFFFFFFF)
    z = x.gather(1, ids).to(torch.float64)
    greedy = t == 0.0
    # (a temperature or a top-p given as a number is the F32 nearest it, as an argument is)
    t = torch.where(greedy, 1.0, t).to(torch.float32).to(torch.float64).unsqueeze(1)
    w = torch.exp((z - z[:, :1]) / t)
    at = torch.arange(vocab, device=x.device)
    first = torch.where(greedy, 1, torch.where(k > 0, k, vocab)).unsqueeze(1)
    w = torch.where(at < first, w, 0.0)
    p = p.to(torch.float32).to(torch.float64).unsqueeze(1)
    before = torch.cumsum(w, 1) - w
    keep = (at < first) & (z > -math.inf) & (w >= mp.to(torch.float32).to(torch.float64).unsqueeze(1))
    keep &= (p >= 1.0) | (before < p * w.sum(1, keepdim=True))
    w = torch.where(keep, w, 0.0)
    run = torch.cumsum(w, 1)
    total = w.sum(1, keepdim=True)
    kept = keep.sum(1, keepdim=True)
    pick = torch.minimum((run <= u.unsqueeze(1) * total).sum(1, keepdim=True), kept - 1)
    return (ids.gather(1, pick).squeeze(1).to(torch.int32), torch.log(w.gather(1, pick) / total).squeeze(1).to(torch.float32),
            kept.squeeze(1).to(torch.int32))


def run(state):
    c = state["c"]
    if own:
        import syntropy_amd.gemv as S
        import syntropy_amd.half as H
        if c["op"] == "product":
            return H.gemv(state["w"], state["x"], c["rows"], act=c["act"], gate=state["gate"], residual=state["residual"],
                          dtype=DT[c["out"]])
        if c["op"] == "norm":
            r = S.block_norm(state["x"], state["branch"], state["g"], EPS, c["rows"], post=state["post"], gate=state["gate"],
                             scale=c["scale"], dtype=DT[c["type"]])
            return r.h, r.y
        r = S.sample_tokens(state["x"], state["u"], **state["how"])
        return r.token, r.logprob, r.kept
    return {"product": _plain_product, "norm": _plain_norm, "sample": _plain_sample}[c["op"]](c, state)


def work(case):
    c = case
    rows = c["rows"]
    if c["op"] == "product":
        es, os = SIZE[c["type"]], SIZE[c["out"]]
        out = rows * c["n"] * (os + (es if c["gate"] else 0) + (os if c["residual"] else 0))
        return {"bytes": es * c["k"] * (c["n"] + rows) + out + (4 * c["n"] if c["bias"] else 0),
                "flops": 2 * c["n"] * c["k"] * rows}
    if c["op"] == "norm":
        es, ss, n = SIZE[c["type"]], SIZE[c["stream"]], c["n"]
        gate = {"none": 0, "channel": n * es, "token": rows * n * es}[c["gate"]]
        # the sum of squares, the norm and the residual sum
        return {"bytes": 2 * rows * n * (es + ss) + gate + 4 * n * (2 if c["post"] else 1),
                "flops": rows * n * (6 + (4 if c["post"] else 0) + (0 if c["gate"] == "none" else 1))}
    # a value is compared, shifted, scaled, exponentiated and added to a sum
    return {"bytes": rows * (c["vocab"] * SIZE[c["type"]] + 16 + (16 if c["each"] else 0)), "flops": 5 * rows * c["vocab"]}


# ---- the same in 64 bits ----------------------------------------------------------------------------

def _exact_product(c, i):
    d = torch.float64
    y = i["x"].to(d) @ i["w"].to(d).T
    if i["bias"] is not None:
        y += i["bias"].to(d)
    act = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
           "gelu": lambda v: v * torch.special.ndtr(v),
           "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[c["act"]]
    y = act(y)
    if i["gate"] is not None:
        y = y * i["gate"].to(d)
    return y if i["residual"] is None else y + i["residual"].to(d)


def _exact_norm(c, i):
    d = torch.float64

    def norm(v, g):
        return g.to(d) * v / (torch.linalg.vector_norm(v, 2, 1, keepdim=True) ** 2 / c["n"] + EPS).sqrt()
    a = i["branch"].to(d)
    a = norm(a, i["post"]) if c["post"] else a
    h = i["x"].to(d) + (c["scale"] * a if i["gate"] is None else c["scale"] * a * i["gate"].to(d))
    return h, norm(h, i["g"])


def _exact_sample(c, i):
    def of(key, r):
        v = i["how"][key]
        return float(v[r]) if torch.is_tensor(v) else float(torch.tensor(v, dtype=torch.float32))
    out = []
    for r in range(c["rows"]):
        z, order = torch.sort(i["x"][r].to(torch.float64), descending=True, stable=True)
        n = int((z > -math.inf).sum())
        temp, k = of("temperature", r), int(of("top_k", r))
        if temp == 0.0:
            temp, k = 1.0, 1
        n = min(n, k) if k > 0 else n
        prob = torch.softmax(z[:n] / temp, 0)
        if of("top_p", r) < 1.0:
            n = min(n, 1 + int((torch.cumsum(prob, 0) < of("top_p", r)).sum()))
        n = min(n, int((prob / prob[0] >= of("min_p", r)).sum()))
        cum = torch.cumsum(prob[:n], 0)
        at = min(int(torch.searchsorted(cum, i["u"][r].to(torch.float64) * cum[-1], right=True)), n - 1)
        out.append((order[at], torch.log(prob[at] / cum[-1]), n))
    return (torch.tensor([int(o[0]) for o in out], dtype=torch.int32, device="cuda"), torch.stack([o[1] for o in out]),
            torch.tensor([o[2] for o in out], dtype=torch.int32, device="cuda"))


def exact(case, seed):
    i = INPUTS[case["op"]](case, seed)
    return {"product": _exact_product, "norm": _exact_norm, "sample": _exact_sample}[case["op"]](case, i)
