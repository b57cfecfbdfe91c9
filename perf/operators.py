"""The token operators as a user's program calls them: sizes, inputs, plain forms and 64-bit values.

Three paths, each with its plain form in elementary torch operations:

connected  a connected layer over int8 weights with a scale for each output channel. Every token
           (row of x) is quantized on the way in: s = amax / 127, code = rint(x * (127 / amax)), both
           in 32 bits, amax at least 2^-100. y = act(s * w_scale * (codes . w) + bias).
score      log probability of each row's given token, the entropy of the row's distribution and its
           `top` most probable tokens (equal logits: the lowest index first), softmax of
           logits / temperature.
grad       the training step of the same: log probabilities and entropies, then the gradient of
           sum(g_logprob * logprob + g_entropy * entropy) with respect to the logits.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_FLOOR = 2.0 ** -100


def listed():
    return [
        # one token through a square projection: a decoding step, where latency is all
        {"name": "connected one token", "kind": "connected", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "act": "linear", "bias": False},
        # a decoding batch through a wide projection: the weights' bytes bound it
        {"name": "connected decode batch", "kind": "connected", "m": 32, "n": 16384, "k": 4096, "dtype": "bf16", "act": "linear", "bias": True},
        # a short prompt in float32 at sizes that fit no tile, with the framework's leaky activation
        {"name": "connected odd", "kind": "connected", "m": 333, "n": 4099, "k": 1003, "dtype": "f32", "act": "leaky", "bias": True},
        # a long prompt or a batch of them: the products bound it
        {"name": "connected long", "kind": "connected", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16", "act": "linear", "bias": False},
        # the distribution after one decoded token, with the alternatives a server reports
        {"name": "score one token", "kind": "score", "rows": 1, "vocab": 131072, "top": 20, "dtype": "bf16", "temperature": 1.0, "masked": 0.0},
        # a decoding batch under a grammar that masks half of an odd vocabulary
        {"name": "score masked batch", "kind": "score", "rows": 48, "vocab": 50001, "top": 5, "dtype": "f32", "temperature": 0.7, "masked": 0.5},
        # the answers of a classifier over the usual 1000 classes
        {"name": "score classes", "kind": "score", "rows": 16384, "vocab": 1000, "top": 5, "dtype": "f16", "temperature": 1.0, "masked": 0.0},
        # every token of a batch of long texts
        {"name": "score long", "kind": "score", "rows": 4096, "vocab": 131072, "top": 20, "dtype": "bf16", "temperature": 1.0, "masked": 0.0},
        # a small training step
        {"name": "grad short", "kind": "grad", "rows": 128, "vocab": 32000, "dtype": "bf16", "temperature": 1.0, "masked": 0.0},
        # float32 logits, an odd vocabulary, some of it masked, at a temperature
        {"name": "grad odd", "kind": "grad", "rows": 777, "vocab": 50001, "dtype": "f32", "temperature": 1.3, "masked": 0.1},
        # a large training step
        {"name": "grad long", "kind": "grad", "rows": 4096, "vocab": 131072, "dtype": "bf16", "temperature": 1.0, "masked": 0.0},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kind = rng.choice(["connected", "score", "grad"])
    if kind == "connected":
        n, k = _spread(rng, 256, 16384), _spread(rng, 256, 16384)
        m = _spread(rng, 1, min(8192, 8192 ** 3 // (n * k)))
        if rng.random() < 0.5:
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        return {"kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "act": rng.choice(["linear", "leaky", "relu"]), "bias": rng.random() < 0.5}
    vocab = _spread(rng, 64, 131072)
    if rng.random() < 0.5:
        vocab = -(-vocab // 16) * 16
    rows = _spread(rng, 1, min(16384, (1 << 28) // vocab))
    case = {"kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": rng.choice([1.0, 0.6, 1.5]), "masked": rng.choice([0.0, 0.0, 0.3])}
    if kind == "score":
        case["top"] = rng.choice([0, 1, 5, 20, 32])
    return case


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    state = {"case": dict(case)}
    if case["kind"] == "connected":
        m, n, k = case["m"], case["n"], case["k"]
        x = torch.randn(m, k, device=dev, generator=g)
        # a few input channels are far larger than the rest, as activations have it
        x *= 1 + 9 * (torch.rand(k, device=dev, generator=g) < 0.01).float()
        state["x"] = x.to(dtype)
        # weight rows are padded to whole 16 bytes, the layout that the layer keeps them in
        codes = torch.zeros(n, -(-k // 16) * 16, device=dev, dtype=torch.int8)
        for i in range(0, n, 4096):
            rows = min(4096, n - i)
            codes[i:i + rows, :k] = torch.randn(rows, k, device=dev, generator=g).mul_(36).round_().clamp_(-127, 127).to(torch.int8)
        state["w"] = codes[:, :k]
        state["w_scales"] = (0.5 + torch.rand(n, device=dev, generator=g)) * (1 / (36 * math.sqrt(k)))
        state["bias"] = torch.randn(n, device=dev, generator=g) if case["bias"] else None
        return state
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.empty(rows, vocab, device=dev, dtype=dtype)
    tokens = torch.empty(rows, device=dev, dtype=torch.int64)
    step = max(1, (1 << 26) // vocab)
    for i in range(0, rows, step):
        part = torch.randn(min(step, rows - i), vocab, device=dev, generator=g)
        # from flat to peaked rows
        part *= 1 + 3 * torch.rand(part.shape[0], 1, device=dev, generator=g)
        if case["masked"]:
            part.masked_fill_(torch.rand(part.shape, device=dev, generator=g) < case["masked"], -math.inf)
        # the given token is mostly a probable one
        noise = 4 * torch.randn(part.shape, device=dev, generator=g)
        tokens[i:i + part.shape[0]] = (part + noise).argmax(-1)
        logits[i:i + part.shape[0]] = part.to(dtype)
    state["logits"], state["tokens"] = logits, tokens
    if case["kind"] == "grad":
        state["g_logprobs"] = -torch.rand(rows, device=dev, generator=g) / rows
        state["g_entropy"] = -0.01 * torch.ones(rows, device=dev) / rows
    return state


# ---- plain forms ------------------------------------------------------------------------------

def _act(y, act):
    if act == "leaky":
        return torch.where(y < 0, y * 0.1, y)
    return torch.where(y > 0, y, y * 0) if act == "relu" else y


def _connected(x, w, w_scales, bias, act):
    v = x.float()
    amax = v.abs().amax(1, keepdim=True).clamp(min=_FLOOR)
    top = torch.full_like(amax, 127.0)
    codes = torch.round(v * (top / amax))
    y = (codes @ w.float().t()) * (amax / top) * w_scales
    if bias is not None:
        y = y + bias
    return _act(y, act).to(x.dtype)


def _distribution(logits, temperature):
    """The log probabilities of every token in 32 bits and the entropies; a row with nothing left has -inf and 0."""
    z = logits.float()
    if temperature != 1.0:
        z = z / temperature
    m = z.amax(1, keepdim=True)
    empty = m == -math.inf
    z = z - torch.where(empty, torch.zeros_like(m), m)
    e = torch.exp(z)
    lp = z - torch.log(e.sum(1, keepdim=True))
    del z, e
    lp = torch.where(empty, torch.full_like(lp, -math.inf), lp)
    p = torch.exp(lp)
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    return lp, p, entropy


def _ordered(logits, top):
    """The indices of each row's largest logits, equal ones by index: whole keys of the order of (value, -index)."""
    bits = logits.float().add(0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    key += torch.arange(logits.shape[1] - 1, -1, -1, device=logits.device)
    return torch.topk(key, top, dim=1).indices


def _score(logits, tokens, top, temperature):
    lp, _, entropy = _distribution(logits, temperature)
    out = {"logprobs": lp.gather(1, tokens[:, None])[:, 0], "entropy": entropy}
    if top:
        out["top_tokens"] = _ordered(logits, top)
        out["top_logprobs"] = lp.gather(1, out["top_tokens"])
    return out


def _grad(logits, tokens, temperature, g_logprobs, g_entropy):
    lp, p, entropy = _distribution(logits, temperature)
    logprobs = lp.gather(1, tokens[:, None])[:, 0]
    inner = torch.where(p > 0, g_logprobs[:, None] + g_entropy[:, None] * (lp + entropy[:, None]), torch.zeros_like(p))
    d = -p * inner
    d.scatter_add_(1, tokens[:, None], g_logprobs[:, None])
    return {"logprobs": logprobs, "entropy": entropy, "grad": (d / temperature).to(logits.dtype)}


# ---- the framework's operators ------------------------------------------------------------------

_kept = {}


def _context():
    """The one context that a program keeps for its GPU."""
    if "context" not in _kept:
        import tensorium_b200
        _kept["context"] = tensorium_b200.Context(torch.cuda.current_device())
    return _kept["context"]


def run(state):
    case = state["case"]
    if case["kind"] == "connected":
        if not own:
            return _connected(state["x"], state["w"], state["w_scales"], state["bias"], case["act"])
        from tensorium_b200.tokens import int8_connected
        return int8_connected(_context(), state["x"], state["w"], state["w_scales"], state["bias"], case["act"])
    temperature = case["temperature"]
    if case["kind"] == "score":
        if not own:
            return _score(state["logits"], state["tokens"], case["top"], temperature)
        from tensorium_b200.tokens import token_logprobs
        r = token_logprobs(_context(), state["logits"], state["tokens"], top=case["top"], temperature=temperature)
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        if case["top"]:
            out["top_tokens"], out["top_logprobs"] = r.top_tokens, r.top_logprobs
        return out
    if not own:
        return _grad(state["logits"], state["tokens"], temperature, state["g_logprobs"], state["g_entropy"])
    from tensorium_b200.tokens import token_logprobs, token_logprobs_backward
    r = token_logprobs(_context(), state["logits"], state["tokens"], temperature=temperature)
    d = token_logprobs_backward(_context(), state["logits"], state["tokens"], r, state["g_logprobs"], state["g_entropy"], temperature=temperature)
    return {"logprobs": r.logprobs, "entropy": r.entropy, "grad": d}


def work(case):
    b = _BYTES[case["dtype"]]
    if case["kind"] == "connected":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * b + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * b, "flops": 2 * m * n * k}
    rows, vocab = case["rows"], case["vocab"]
    if case["kind"] == "score":
        # a product, an exponential and two sums for each logit
        return {"bytes": rows * (vocab * b + 8 + 8 + case["top"] * 12), "flops": 5 * rows * vocab}
    return {"bytes": rows * (2 * vocab * b + 8 + 8 + 8), "flops": 11 * rows * vocab}


# ---- 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "connected":
        x, w = state["x"].double(), state["w"]
        largest = torch.clamp(torch.max(torch.abs(x), 1).values, min=_FLOOR)
        # the codes are whole numbers that the definition takes from 32-bit arithmetic: a quotient
        # and a product of two 32-bit numbers, each rounded once (both are exact enough in 64 bits)
        factor = (127.0 / largest).float().double()
        codes = torch.round((x * factor[:, None]).float().double())
        y = torch.empty(case["m"], case["n"], device=x.device, dtype=torch.float64)
        for i in range(0, case["n"], 4096):
            y[:, i:i + 4096] = codes @ w[i:i + 4096].double().t()
        y *= torch.outer(largest / 127.0, state["w_scales"].double())
        if state["bias"] is not None:
            y += state["bias"].double()
        slope = {"linear": 1.0, "leaky": 0.1, "relu": 0.0}[case["act"]]
        return torch.where(y < 0, y * slope, y)
    temperature, tokens = case["temperature"], state["tokens"]
    found = {"logprobs": [], "entropy": [], "top_tokens": None, "top_logprobs": [], "grad": []}
    step = max(1, (1 << 27) // case["vocab"])
    for i in range(0, case["rows"], step):
        z = state["logits"][i:i + step].double() / temperature
        t = tokens[i:i + step]
        at = torch.arange(len(t), device=t.device)
        lp = z - torch.logsumexp(z, 1)[:, None]
        lp[torch.isneginf(z)] = -math.inf
        p = lp.exp()
        h = -torch.xlogy(p, p).sum(1)
        found["logprobs"].append(lp[at, t])
        found["entropy"].append(h)
        if case["kind"] == "score":
            if case["top"]:
                found["top_logprobs"].append(torch.topk(lp, case["top"]).values)
            continue
        a, b = state["g_logprobs"][i:i + step].double(), state["g_entropy"][i:i + step].double()
        # d logprob / dz = onehot - p, d entropy / dz = -p (log p + entropy)
        d = -a[:, None] * p - b[:, None] * (torch.xlogy(p, p) + p * h[:, None])
        d[at, t] += a
        found["grad"].append(d / temperature)
    if case["kind"] == "grad":
        return {k: torch.cat(found[k]) for k in ("logprobs", "entropy", "grad")}
    out = {k: torch.cat(found[k]) for k in ("logprobs", "entropy")}
    if case["top"]:
        out["top_tokens"], out["top_logprobs"] = None, torch.cat(found["top_logprobs"])
    return out
