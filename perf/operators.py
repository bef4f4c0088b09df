"""Cases, inputs, plain forms and exact results of the sequence operators of keops_amd.torch.

Three operators, each with the passes that a program makes of it:

  attention   bucket_attention: softmax attention with a learned bias by buckets of the relative position
              (forward over a prompt, one token against a cache, forward + backward)
  decay       decay_attention / decay_attention_step: linear attention with a decay for each head
              (forward over a prompt, one token against the state, forward + backward)
  logprobs    token_logprobs: log probabilities of given tokens, entropy and top alternatives of rows of logits
              (forward, forward + backward)

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the framework's calls.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    def attention(name, what, batch, heads, kv_heads, queries, keys, dim, dtype, causal, ragged, both, buckets=32, reach=128):
        return {"name": name, "op": "attention", "what": what, "batch": batch, "heads": heads, "kv_heads": kv_heads,
                "queries": queries, "keys": keys, "dim": dim, "dtype": dtype, "causal": causal, "ragged": ragged,
                "both": both, "buckets": buckets, "reach": reach}

    def decay(name, what, batch, heads, kv_heads, tokens, dim, dim_v, dtype, ragged, start):
        return {"name": name, "op": "decay", "what": what, "batch": batch, "heads": heads, "kv_heads": kv_heads,
                "tokens": tokens, "dim": dim, "dim_v": dim_v, "dtype": dtype, "ragged": ragged, "start": start}

    def logprobs(name, what, rows, vocab, dtype, top):
        return {"name": name, "op": "logprobs", "what": what, "rows": rows, "vocab": vocab, "dtype": dtype, "top": top}

    return [
        # one new token of a small batch against short caches: latency
        attention("attention token short", "token", 4, 8, 8, 1, 300, 64, "bf16", True, True, False),
        # one new token of a full serving batch, caches of different lengths
        attention("attention token batch", "token", 32, 8, 8, 1, 2048, 64, "bf16", True, True, False),
        # one new token of a single long document, shared key/value heads
        attention("attention token long", "token", 1, 16, 2, 1, 131072, 128, "fp16", True, False, False),
        # a long prompt, causal
        attention("attention prompt", "forward", 1, 8, 8, 16384, 16384, 128, "bf16", True, False, False),
        # a training step's attention layer (the shape of the softmax benchmark of this repository)
        attention("attention train", "train", 4, 8, 8, 4096, 4096, 64, "bf16", True, False, False),
        # an encoder-decoder style layer in full precision: ragged keys, both directions, odd sizes
        attention("attention train odd", "train", 3, 6, 3, 517, 777, 40, "fp32", False, True, True),
        # one new token of a serving batch against its states
        decay("decay token batch", "token", 64, 16, 16, 1, 128, 128, "bf16", False, True),
        # a long prompt, final state kept for the tokens that follow
        decay("decay prompt", "forward", 1, 16, 16, 16384, 128, 128, "bf16", False, False),
        # a training step's layer
        decay("decay train", "train", 4, 8, 8, 4096, 64, 64, "bf16", False, False),
        # a continued, padded batch in full precision, shared key/value heads, odd sizes
        decay("decay train odd", "train", 3, 6, 2, 777, 40, 72, "fp32", True, True),
        # the logits of a few sequences that generate, with alternatives for the answer
        logprobs("logprobs token", "forward", 4, 32003, "bf16", 5),
        # a policy update: log probabilities and entropies with gradients, odd vocabulary
        logprobs("logprobs train", "train", 2048, 50021, "fp32", 0),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    most_flops = max(work(c)["flops"] for c in listed())
    most_bytes = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["attention", "attention", "decay", "decay", "logprobs"])
        if op == "attention":
            what = rng.choice(["token", "forward", "train"])
            groups, kv = rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 8])
            both = rng.random() < 0.4 and what != "token"
            case = {"op": op, "what": what, "batch": _log_int(rng, 1, 32), "heads": groups * kv, "kv_heads": kv,
                    "queries": 1 if what == "token" else _log_int(rng, 2, 4096),
                    "keys": _log_int(rng, 1, 131072 if what == "token" else 4096),
                    "dim": rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128, 128]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    "causal": what == "token" or (not both and rng.random() < 0.7), "ragged": rng.random() < 0.5, "both": both,
                    "buckets": rng.choice([16, 32, 64]), "reach": rng.choice([64, 128, 200, 512])}
            if case["causal"] and what != "token":
                case["keys"] = max(case["keys"], case["queries"])
        elif op == "decay":
            what = rng.choice(["token", "forward", "train"])
            groups, kv = rng.choice([1, 1, 2, 3, 4]), rng.choice([1, 2, 4, 8, 16])
            case = {"op": op, "what": what, "batch": _log_int(rng, 1, 64), "heads": groups * kv, "kv_heads": kv,
                    "tokens": 1 if what == "token" else _log_int(rng, 2, 8192), "dim": rng.choice([16, 32, 40, 64, 64, 96, 128, 128]),
                    "dim_v": rng.choice([16, 32, 64, 64, 72, 128, 128]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    "ragged": what != "token" and rng.random() < 0.5, "start": what == "token" or rng.random() < 0.5}
        else:
            case = {"op": op, "what": rng.choice(["forward", "train"]), "rows": _log_int(rng, 1, 4096), "vocab": _log_int(rng, 500, 200000),
                    "dtype": rng.choice(["bf16", "fp16", "fp32"]), "top": rng.choice([0, 1, 5, 20])}
        w = work(case)
        # the plain forms hold (batch, heads, queries, keys) tables: those stay below 2^31 entries
        table = {"attention": lambda: case["batch"] * case["heads"] * case["queries"] * case["keys"],
                 "decay": lambda: case["batch"] * case["heads"] * case["tokens"] ** 2, "logprobs": lambda: 0}[op]()
        if w["flops"] <= most_flops and w["bytes"] <= most_bytes and table <= 1 << 31:
            return case


def _lengths(case, longest):
    """Lengths of a padded batch: from about a third of the longest to all of it."""
    if not case["ragged"]:
        return None
    b = case["batch"]
    return [max(1, longest - (longest * 2 * i) // (3 * b)) for i in range(b)]


# ---------------------------------------------------------------------------------------------------- work
def _pairs(case):
    """(query, key) pairs of one head, summed over the batch."""
    lens = _lengths(case, case["keys"]) or [case["keys"]] * case["batch"]
    m = case["queries"]
    if not case["causal"] or case["what"] == "token":
        return sum(m * n for n in lens)
    first = case["keys"] - m  # key position of the first query
    total = 0
    for n in lens:  # row i sees min(first + i + 1, n) keys
        full = max(0, min(m, n - first))
        total += full * (first + 1) + full * (full - 1) // 2 + (m - full) * n
    return total


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "attention":
        lens = _lengths(case, case["keys"]) or [case["keys"]] * case["batch"]
        rows = case["batch"] * case["heads"] * case["queries"] * case["dim"] * e
        cols = sum(lens) * case["kv_heads"] * case["dim"] * e
        table = case["heads"] * case["buckets"] * 4
        flops = 4.0 * _pairs(case) * case["heads"] * case["dim"]
        if case["what"] == "train":  # seven products; q, k, v, the output's gradient in; the output and four gradients out
            return {"bytes": float(4 * rows + 4 * cols + 2 * table), "flops": 3.5 * flops}
        return {"bytes": float(2 * rows + 2 * cols + table), "flops": flops}
    if case["op"] == "decay":
        lens = _lengths(case, case["tokens"]) or [case["tokens"]] * case["batch"]
        t, h, kv, d, dv = sum(lens), case["heads"], case["kv_heads"], case["dim"], case["dim_v"]
        state = case["batch"] * h * d * dv * 4
        one = t * (h * (d + dv) + kv * (d + dv)) * e
        states = state * ((2 if case["start"] else 1) if case["what"] != "train" else (4 if case["start"] else 2))
        flops = 4.0 * t * h * d * dv
        # forward: q, k, v in, output out; training: the output's gradient in and three gradients out too
        return {"bytes": float((2 if case["what"] == "train" else 1) * one + states), "flops": (3.0 if case["what"] == "train" else 1.0) * flops}
    n = case["rows"] * case["vocab"]
    train = case["what"] == "train"
    return {"bytes": float(n * e * (2 if train else 1) + case["rows"] * (24 + 12 * case["top"])), "flops": float(n * (8 if train else 5))}


# ---------------------------------------------------------------------------------------------------- inputs
def _decays(heads):
    """log of the decay of each head: windows of about 2 to 1000 tokens, spread over the heads."""
    e = torch.linspace(1.0, 10.0, heads, dtype=torch.float64) if heads > 1 else torch.tensor([5.0], dtype=torch.float64)
    return torch.log1p(-torch.exp2(-e)).float()


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=gen) * scale).to(dtype)

    train = case["what"] == "train"
    s = {"case": dict(case)}
    if case["op"] == "attention":
        b, h, kv, m, n, d = (case[x] for x in ("batch", "heads", "kv_heads", "queries", "keys", "dim"))
        # projections as a layer leaves them: (batch, position, head, dim), seen as (batch, head, position, dim)
        s["q"] = normal(b, m, h, d).transpose(1, 2)
        s["k"] = normal(b, n, kv, d).transpose(1, 2)
        s["v"] = normal(b, n, kv, d).transpose(1, 2)
        if case["what"] == "token":  # a cache is laid out by head
            s["k"], s["v"] = s["k"].contiguous(), s["v"].contiguous()
        s["bias"] = normal(h, case["buckets"], dtype=torch.float32)
        lens = _lengths(case, n)
        s["lengths"] = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
        # a new token comes after its cache; the queries of a causal block are its last positions
        if case["what"] == "token":
            s["first"] = n - 1 if lens is None else s["lengths"] - 1
        else:
            s["first"] = n - m if case["causal"] else 0
        s["borders"] = torch.tensor(_borders(case["buckets"], case["reach"], case["both"]), device=dev)
        if own:
            from keops_amd.torch import PositionBuckets

            s["buckets"] = PositionBuckets(case["buckets"], case["reach"], bidirectional=case["both"])
        leaves = ("q", "k", "v", "bias")
        if train:
            s["grad"] = normal(b, m, h, d).transpose(1, 2)
    elif case["op"] == "decay":
        b, h, kv, t, d, dv = (case[x] for x in ("batch", "heads", "kv_heads", "tokens", "dim", "dim_v"))
        s["q"] = normal(b, t, h, d).transpose(1, 2)
        s["k"] = normal(b, t, kv, d, scale=d ** -0.5).transpose(1, 2)
        s["v"] = normal(b, t, kv, dv).transpose(1, 2)
        s["log_decay"] = _decays(h).to(dev)
        s["state"] = normal(b, h, d, dv, dtype=torch.float32) if case["start"] else None
        lens = _lengths(case, t)
        s["lengths"] = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
        leaves = ("q", "k", "v") + (("state",) if case["start"] else ())
        if case["what"] == "token":
            s["q"], s["k"], s["v"] = (s[x][:, :, 0] for x in ("q", "k", "v"))
        if train:
            s["grad"] = normal(b, t, h, dv).transpose(1, 2)
            s["grad_state"] = normal(b, h, d, dv, dtype=torch.float32)
    else:
        r, v = case["rows"], case["vocab"]
        s["logits"] = normal(r, v, scale=3.0)
        s["tokens"] = torch.randint(0, v, (r,), device=dev, generator=gen)
        leaves = ("logits",)
        if train:
            s["grad"] = normal(r, dtype=torch.float32)
            s["grad_entropy"] = normal(r, dtype=torch.float32, scale=0.1)
            s["grad_top"] = normal(r, case["top"], dtype=torch.float32, scale=0.1)
    if train:
        for x in leaves:
            s[x].requires_grad_(True)
    s["leaves"] = leaves
    return s


def _borders(buckets, reach, both):
    """Smallest distances of the buckets after the first one, for one direction: one bucket for each of the first
    distances, the rest in equal steps of the logarithm up to ``reach``.  Whole numbers throughout: bucket ``near + t``
    begins at the smallest n with (n / near)^(count - near) >= (reach / near)^t."""
    count = buckets // 2 if both else buckets
    near = count // 2
    steps = count - near
    out = list(range(1, near + 1))
    for t in range(1, steps):
        n = out[-1]
        while n ** steps < near ** (steps - t) * reach ** t:
            n += 1
        out.append(n)
    return out


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    op, what = case["op"], case["what"]
    forward = {"attention": _attention, "decay": _decay, "logprobs": _logprobs}[op]
    if what != "train":
        with torch.no_grad():
            return forward(state, state)
    if own:
        inputs = state
    else:  # gradients in 32 bits, rounded once at the end
        inputs = dict(state)
        for x in state["leaves"]:
            inputs[x] = state[x].detach().float().requires_grad_(True)
    with torch.enable_grad():
        out = forward(state, inputs)
    leaves = [inputs[x] for x in state["leaves"]]
    if op == "attention":
        outs, seeds = [out["out"]], [state["grad"]]
    elif op == "decay":
        outs, seeds = [out["out"], out["state"]], [state["grad"], state["grad_state"]]
    else:
        outs, seeds = [out["logprob"], out["entropy"]], [state["grad"], state["grad_entropy"]]
        if case["top"]:
            outs, seeds = outs + [out["top_logprob"]], seeds + [state["grad_top"]]
    if not own:  # the rounded output is what the caller sees; the gradient flows through its 32-bit form
        seeds = [g.to(o.dtype) for g, o in zip(seeds, outs)]
    grads = torch.autograd.grad(outs, leaves, seeds)
    result = {k: t.detach() for k, t in out.items()}
    for x, g in zip(state["leaves"], grads):
        result["grad_" + x] = g
    if not own:
        result = {k: _round(state, k, t) for k, t in result.items()}
    return result


def _round(state, key, t):
    if key.startswith("grad_"):
        return t.to(state[key[5:]].dtype)
    if key == "out":
        return t.to(state["q"].dtype)
    return t


def _attention(state, x):
    case = state["case"]
    scale = case["dim"] ** -0.5
    if own:
        from keops_amd.torch import bucket_attention

        return {"out": bucket_attention(x["q"], x["k"], x["v"], x["bias"], state["buckets"], causal=case["causal"],
                                        key_lengths=state["lengths"], query_start=state["first"], scale=scale)}
    q, k, v, bias = (x[n].float() for n in ("q", "k", "v", "bias"))
    b, h, m, d = q.shape
    kv, n = k.shape[1], k.shape[2]
    q = q.reshape(b, kv, h // kv, m, d)
    scores = (q.reshape(b, kv, -1, d) @ k.transpose(-1, -2).contiguous()).view(b, kv, h // kv, m, n) * scale
    first = state["first"]
    rows = torch.arange(m, device=q.device)
    cols = torch.arange(n, device=q.device)
    first = first.long().view(b, 1, 1) if torch.is_tensor(first) else first
    away = cols - (rows[:, None] + first)  # (m, n) or (b, m, n)
    # bucket of every distance that occurs, then one table of biases by distance
    low, high = -(m + n + 1), n + m + 1
    dist = torch.arange(low, high + 1, device=q.device)
    gone = (dist.abs() if case["both"] else (-dist).clamp(min=0))
    bucket = (gone[:, None] >= state["borders"]).sum(-1)
    if case["both"]:
        bucket = bucket + (dist > 0) * (case["buckets"] // 2)
    by_distance = bias[:, bucket].view(kv, h // kv, -1)
    added = by_distance[:, :, away - low]  # (kv, g, m, n) or (kv, g, b, m, n)
    scores = scores + (added.permute(2, 0, 1, 3, 4) if added.dim() == 5 else added)
    seen = torch.ones_like(away, dtype=torch.bool)
    if case["causal"]:
        seen = away <= 0
    if state["lengths"] is not None:
        seen = seen & (cols < state["lengths"].long().view(b, 1, 1))
    seen = seen.view(-1, 1, 1, m, n)
    scores = torch.where(seen, scores, scores.new_full((), -math.inf))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = (p.view(b, kv, -1, n) @ v).view(b, h, m, d)
    return {"out": out if case["what"] == "train" else out.to(state["q"].dtype)}


def _decay(state, x):
    case = state["case"]
    scale = case["dim"] ** -0.5
    if own:
        from keops_amd.torch import decay_attention, decay_attention_step

        if case["what"] == "token":
            return {"out": decay_attention_step(x["q"], x["k"], x["v"], x["log_decay"], x["state"], scale=scale), "state": x["state"]}
        out, last = decay_attention(x["q"], x["k"], x["v"], x["log_decay"], initial_state=x["state"], lengths=state["lengths"], scale=scale)
        return {"out": out, "state": last}
    q, k, v = (x[n].float() for n in ("q", "k", "v"))
    log_decay, start = x["log_decay"], x["state"]
    if case["what"] == "token":
        g = q.shape[1] // k.shape[1]
        k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        new = start * torch.exp(log_decay)[None, :, None, None] + k[..., :, None] * v[..., None, :]
        out = (q[..., None] * new).sum(-2) * scale
        return {"out": out.to(state["q"].dtype), "state": start.copy_(new)}
    b, h, t, d = q.shape
    g = h // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    pos = torch.arange(t, device=q.device)
    size = torch.full((b,), t, device=q.device) if state["lengths"] is None else state["lengths"].long()
    there = (pos < size[:, None]).float()[:, None, :, None]  # (b, 1, t, 1)
    away = pos[:, None] - pos
    weights = torch.where(away >= 0, torch.exp(away.clamp(min=0) * log_decay[:, None, None]), torch.zeros((), device=q.device))
    q, k, v = q * there, k * there, v * there
    out = ((q @ k.transpose(-1, -2).contiguous()) * weights) @ v
    left = (size[:, None, None] - 1 - pos).clamp(min=0) * log_decay[:, None]  # (b, h, t)
    last = (k * torch.exp(left)[..., None]).transpose(-1, -2).contiguous() @ v
    if start is not None:
        out = out + (q @ start) * torch.exp((pos + 1) * log_decay[:, None])[None, :, :, None]
        last = last + start * torch.exp(size[:, None] * log_decay)[..., None, None]
    out = out * scale
    return {"out": out if case["what"] == "train" else out.to(state["q"].dtype), "state": last}


def _logprobs(state, x):
    case = state["case"]
    if own:
        from keops_amd.torch import token_logprobs

        r = token_logprobs(x["logits"], state["tokens"], top=case["top"])
        return {"logprob": r.logprob, "entropy": r.entropy, "top_logprob": r.top_logprob, "top_index": r.top_index}
    z = x["logits"].float()
    z = z - z.detach().amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    logprob = (z.gather(-1, state["tokens"][:, None]) - log_total)[:, 0]
    entropy = log_total[:, 0] - (e * z).sum(-1) / total[:, 0]
    # equal values: the lowest index first.  One whole number for each value, by value and then by index
    bits = (x["logits"].detach().float() + 0.0).view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    index = torch.arange(z.shape[-1], device=z.device)
    key = order * (1 << 24) + (z.shape[-1] - 1 - index)
    best = z.shape[-1] - 1 - (key.topk(case["top"], -1).values & ((1 << 24) - 1))
    return {"logprob": logprob, "entropy": entropy, "top_logprob": z.gather(-1, best) - log_total, "top_index": best}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "decay": _exact_decay, "logprobs": _exact_logprobs}[case["op"]](case, s)


def _bucket_of(case, away):
    """Bucket of the key that lies ``away`` positions after the query."""
    count = case["buckets"] // 2 if case["both"] else case["buckets"]
    base = count if case["both"] and away > 0 else 0
    n = abs(away) if case["both"] else max(0, -away)
    near = count // 2
    if n < near:
        return base + n
    t = 0
    while t + 1 < count - near and n ** (count - near) >= near ** (count - near - t - 1) * case["reach"] ** (t + 1):
        t += 1
    return base + near + t


def _exact_attention(case, s):
    """One head of one sequence at a time, rows in blocks."""
    train = case["what"] == "train"
    b, h, m, d = s["q"].shape
    n, g = s["k"].shape[2], h // s["k"].shape[1]
    dev, scale = s["q"].device, d ** -0.5
    reach = max(case["reach"], case["buckets"]) + 1
    table = torch.tensor([_bucket_of(case, a) for a in range(-reach, reach + 1)], device=dev)
    lens = [n] * b if s["lengths"] is None else s["lengths"].tolist()
    first = s["first"].tolist() if torch.is_tensor(s["first"]) else [s["first"]] * b
    out = torch.zeros(b, h, m, d, dtype=torch.float64, device=dev)
    dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device=dev) for x in (s["q"], s["k"], s["v"]))
    db = torch.zeros(h, case["buckets"], dtype=torch.float64, device=dev)
    for i in range(b):
        end = lens[i]
        for j in range(h):
            k, v = s["k"][i, j // g, :end].double(), s["v"][i, j // g, :end].double()
            for r in range(0, m, 4096):
                q = s["q"][i, j, r:r + 4096].double()
                at = first[i] + r + torch.arange(q.shape[0], device=dev)
                away = torch.arange(end, device=dev)[None] - at[:, None]
                bucket = table[away.clamp(-reach, reach) + reach]
                z = q @ k.t() * scale + s["bias"][j].double()[bucket]
                if case["causal"]:
                    z = z.masked_fill(away > 0, -math.inf)
                p = torch.softmax(z, -1).nan_to_num(0.0)
                o = p @ v
                out[i, j, r:r + 4096] = o
                if not train:
                    continue
                go = s["grad"][i, j, r:r + 4096].double()
                ds = p * (go @ v.t() - (go * o).sum(-1, keepdim=True))
                dq[i, j, r:r + 4096] = ds @ k * scale
                dk[i, j // g, :end] += ds.t() @ q * scale
                dv[i, j // g, :end] += p.t() @ go
                db[j].index_add_(0, bucket.reshape(-1), ds.reshape(-1))
    return {"out": out, "grad_q": dq, "grad_k": dk, "grad_v": dv, "grad_bias": db} if train else {"out": out}


def _exact_decay(case, s):
    """The recurrence, one token after the other."""
    h, scale = case["heads"], case["dim"] ** -0.5
    gamma = torch.exp(s["log_decay"].double())[None, :, None, None]
    q, k, v = (s[x].double() for x in ("q", "k", "v"))
    if case["what"] == "token":
        q, k, v = q[:, :, None], k[:, :, None], v[:, :, None]
    g = h // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    b, _, t, d = q.shape
    size = torch.full((b,), t, device=q.device) if s["lengths"] is None else s["lengths"].long()
    size = size.view(b, 1, 1, 1)
    S = s["state"].double() if s["state"] is not None else torch.zeros(b, h, d, v.shape[-1], dtype=torch.float64, device=q.device)
    train = case["what"] == "train"
    go = s["grad"].double() if train else None
    out, dq, dk, dv = (torch.zeros_like(x) for x in (v, q, k, v))
    for i in range(t):
        S = torch.where(i < size, gamma * S + k[:, :, i, :, None] * v[:, :, i, None, :], S)
        live = (i < size)[..., 0]
        out[:, :, i] = (q[:, :, i, None] @ S)[:, :, 0] * scale * live
        if train:
            dq[:, :, i] = (S @ go[:, :, i, :, None])[..., 0] * scale * live
    if not train:
        return {"out": out[:, :, 0] if case["what"] == "token" else out, "state": S}
    R = s["grad_state"].double()
    for i in reversed(range(t)):
        live = i < size
        R = torch.where(live, R + q[:, :, i, :, None] * go[:, :, i, None, :] * scale, R)
        dk[:, :, i] = (R @ v[:, :, i, :, None])[..., 0] * live[..., 0]
        dv[:, :, i] = (k[:, :, i, None] @ R)[:, :, 0] * live[..., 0]
        R = torch.where(live, gamma * R, R)
    dk, dv = (x.view(b, h // g, g, t, -1).sum(2) for x in (dk, dv))
    res = {"out": out, "state": S, "grad_q": dq, "grad_k": dk, "grad_v": dv}
    if s["state"] is not None:
        res["grad_state"] = R
    return res


def _exact_logprobs(case, s):
    """Rows in blocks."""
    k = case["top"]
    parts = []
    for r in range(0, case["rows"], 512):
        z = s["logits"][r:r + 512].double()
        tok = s["tokens"][r:r + 512, None]
        lp = torch.log_softmax(z, -1)
        p = lp.exp()
        ent = -(p * lp).sum(-1)
        best = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]
        part = {"logprob": lp.gather(-1, tok)[:, 0], "entropy": ent, "top_logprob": lp.gather(-1, best), "top_index": best}
        if case["what"] == "train":
            a, ge = s["grad"][r:r + 512, None].double(), s["grad_entropy"][r:r + 512, None].double()
            gt = s["grad_top"][r:r + 512].double()
            dz = -p * (a + gt.sum(-1, keepdim=True)) - ge * p * (lp + ent[:, None])
            dz.scatter_add_(-1, tok, a)
            dz.scatter_add_(-1, best, gt)
            part["grad_logits"] = dz
        parts.append(part)
    return {x: torch.cat([p[x] for p in parts]) for x in parts[0]}
