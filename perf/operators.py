"""What the operators around the logits and the packed batch cost: cases, their
inputs, one pass in plain torch operations and one through this package.

  token_logprobs   log probabilities of given tokens, the entropy, and the top
                   alternatives of every position; its gradient
  distillation     the divergence from a teacher's top logits, with the hard
                   targets' cross-entropy beside it; its gradient
  span_attention   attention within documents packed into one row, prompts
                   seen in both directions; its gradient

Vocabularies, head counts and sequence lengths are those of this package's
model configurations, with odd ones between them.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------- cases --

def _logprobs(name, rows, vocab, top, dtype="bf16", temperature=1.0, grad=False, pad=0):
    return {"name": name, "op": "token_logprobs", "rows": rows, "vocab": vocab, "pad": pad,
            "top": top, "dtype": dtype, "temperature": temperature, "grad": grad}


def _distill(name, rows, vocab, k, dtype="bf16", temperature=1.0, hard=True, grad=True, pad=0,
             compact=False):
    return {"name": name, "op": "distillation", "rows": rows, "vocab": vocab, "pad": pad, "k": k,
            "dtype": dtype, "temperature": temperature, "hard": hard, "grad": grad,
            "compact": compact}


def _attention(name, batch, seq, heads, kv_heads, dim, docs, prefix=0.0, tail=0, grad=False):
    return {"name": name, "op": "span_attention", "batch": batch, "seq": seq, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "docs": docs, "prefix": prefix, "tail": tail,
            "grad": grad}


def listed():
    return [
        # The alternatives of one position, as a caller inspecting a model asks for them.
        _logprobs("logprobs_one", 1, 151936, 20),
        # The answers' tokens of a small batch of multiple-choice questions, sampled at 0.7.
        _logprobs("logprobs_few", 67, 128256, 5, temperature=0.7),
        # A teacher's pass over a batch: four sequences of 1024, alternatives kept for each.
        _logprobs("logprobs_teacher", 4 * 1023, 151936, 64),
        # Evaluation from f32 logits of an odd vocabulary in padded rows, no alternatives.
        _logprobs("logprobs_odd_f32", 777, 32003, 0, dtype="f32", pad=61),
        # A policy's training step: gradients through log probability and entropy.
        _logprobs("logprobs_train", 2 * 1023, 128256, 0, grad=True),
        # A short ragged batch of a small vocabulary: launches count.
        _distill("distill_small", 31, 1024, 8, temperature=2.0),
        # The students' training step on stored teacher alternatives and the hard targets.
        _distill("distill_train", 2 * 1023, 128256, 64, temperature=2.0, compact=True),
        # Another vocabulary, odd row count, the divergence alone.
        _distill("distill_soft", 511, 151936, 20, hard=False),
        # A short packed row of a small model.
        _attention("packed_small", 1, 200, 4, 2, 64, docs=3, tail=9),
        # Training on eight packed rows of 512, short documents.
        _attention("packed_short_train", 8, 512, 14, 2, 64, docs=5, tail=17, grad=True),
        # Training on four packed rows of 2048 with prompts seen in both directions.
        _attention("packed_train", 4, 2048, 32, 8, 128, docs=6, prefix=0.25, grad=True),
        # A teacher's pass over one long row: two dozen documents of very different lengths.
        _attention("packed_long", 1, 8191, 32, 8, 128, docs=7, tail=100),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["token_logprobs", "distillation", "span_attention"])
    if op == "span_attention":
        heads, kv_heads, dim = rng.choice([(4, 2, 64), (14, 2, 64), (32, 8, 128), (8, 1, 128),
                                           (6, 6, 64)])
        seq = _log_int(rng, 1, 8191)
        # Where every document is one token, dq and dk are zero and only rounding is left.
        grad = rng.random() < 0.5 and 16 <= seq <= 4096
        most = (4 * 32 * 2048 ** 2 if grad else 32 * 8191 ** 2) // (heads * seq * seq)
        batch = _log_int(rng, 1, max(1, min(16, most)))
        tail = rng.randrange(0, seq // 4 + 1)
        docs = min(_log_int(rng, 1, 40), max(1, (seq - tail) // (4 if grad else 1)))
        return _drop_name(_attention("", batch, seq, heads, kv_heads, dim, docs,
                                     rng.choice([0.0, 0.1, 0.5]), tail, grad))
    vocab = _log_int(rng, 300, 151936)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    grad = rng.random() < 0.5
    most = (2046 * 128256 if grad or op == "distillation" else 4092 * 151936) // vocab
    if dtype == "f32":
        most //= 2
    rows = _log_int(rng, 1, min(most, 4092))
    pad = rng.choice([0, 0, 5, 64, 128])
    temperature = rng.choice([1.0, 1.0, 0.6, 1.7])
    k = rng.choice([1, 3, 8, 20, 50, 64, 128])
    if op == "token_logprobs":
        return _drop_name(_logprobs("", rows, vocab, 0 if grad else rng.choice([0, k, k]), dtype,
                                    temperature, grad, pad))
    return _drop_name(_distill("", rows, vocab, k, dtype, temperature, rng.random() < 0.6, grad,
                               pad, rng.random() < 0.5))


def _drop_name(case):
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs --

def _lengths(case):
    """The documents' lengths in one row: the case's own, in an order that the seed gives."""
    total, docs = case["seq"] - case["tail"], case["docs"]
    rng = random.Random(1000 * case["seq"] + docs)
    weight = [rng.uniform(0.1, 1.0) ** 2 for _ in range(docs)]
    cuts = [round(total * sum(weight[:i]) / sum(weight)) for i in range(docs + 1)]
    return [b - a for a, b in zip(cuts, cuts[1:]) if b > a]


def _prefix_of(case, length):
    return int(case["prefix"] * length)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] == "span_attention":
        return _prepare_attention(case, seed, g)
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    logits = torch.randn(rows, vocab + case["pad"], device="cuda", generator=g)
    logits *= 2.0
    # What a trained model's row looks like: a few dozen tokens well above the rest.
    likely = torch.randint(0, vocab, (rows, 40), device="cuda", generator=g)
    height = 4.0 + 3.0 * torch.randn(rows, 40, device="cuda", generator=g)
    logits.scatter_add_(1, likely, height)
    logits += 3.0 * torch.randn(rows, 1, device="cuda", generator=g)
    # Tokens that the caller ruled out.
    out = torch.randint(0, vocab, (rows, 4), device="cuda", generator=g)
    logits.scatter_(1, out, float("-inf"))
    state = {"case": case, "logits": logits.to(dtype)[:, :vocab]}
    del logits
    # Given tokens: mostly likely ones, some any, some padding.
    pick = torch.randint(0, 40, (rows, 1), device="cuda", generator=g)
    tokens = likely.gather(1, pick).squeeze(1)
    tokens = torch.where((tokens[:, None] == out).any(1), (out[:, 0] + 1) % vocab, tokens)
    lost = state["logits"].gather(1, tokens[:, None]).squeeze(1) == float("-inf")
    skipped = torch.rand(rows, device="cuda", generator=g) < 0.05
    state["tokens"] = torch.where(lost | (skipped & (rows > 1)), -1, tokens)
    if case["op"] == "token_logprobs":
        if case["grad"]:
            state["d_logprobs"] = torch.randn(rows, device="cuda", generator=g) / rows
            state["d_entropy"] = torch.randn(rows, device="cuda", generator=g) / rows * 0.1
        return state
    k = case["k"]
    # Distinct alternatives: every row steps through the vocabulary from a place of its own.
    step = max(1, vocab // k)
    first = torch.randint(0, step, (rows, 1), device="cuda", generator=g)
    ids = first + step * torch.randperm(k, device="cuda", generator=g)[None, :]
    ids = ids % vocab
    fall = torch.rand(rows, k, device="cuda", generator=g).cumsum(1) * (8.0 / k)
    heights = 9.0 - fall - 2.0 * torch.rand(rows, 1, device="cuda", generator=g)
    own_logits = state["logits"].gather(1, ids)
    lost = own_logits == float("-inf")
    state["logits"].scatter_(1, ids, torch.where(
        lost, 0.0, heights + torch.randn(rows, k, device="cuda", generator=g)).to(dtype))
    # Some rows hold fewer alternatives than the others.
    fewer = torch.rand(rows, 1, device="cuda", generator=g) < 0.1
    ids = torch.where(fewer & (torch.arange(k, device="cuda")[None, :] >= (k + 1) // 2), -1, ids)
    if case["compact"]:
        state["teacher_ids"] = ids.to(torch.int32)
        state["teacher_logits"] = heights.to(torch.bfloat16)
    else:
        state["teacher_ids"] = ids
        state["teacher_logits"] = heights - heights.exp().sum(1, keepdim=True).log() - 0.1
    if case["grad"]:
        state["d_kl"] = (0.5 + torch.rand(rows, device="cuda", generator=g)) / rows
        state["d_ce"] = (0.5 + torch.rand(rows, device="cuda", generator=g)) / rows
    return state


def _prepare_attention(case, seed, g):
    b, s, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))

    def normal(heads, gain=1.0):
        x = torch.randn(b, s, heads, d, device="cuda", generator=g)
        return (x * gain).to(torch.bfloat16)

    rng = np.random.default_rng(seed)
    documents = np.full((b, s), -1, dtype=np.int32)
    prefix = np.zeros((b, s), dtype=np.int32)
    for row in range(b):
        at = 0
        for n, length in enumerate(rng.permutation(_lengths(case))):
            documents[row, at:at + length] = n
            prefix[row, at:at + length] = _prefix_of(case, int(length))
            at += length
    state = {"case": case, "q": normal(h, 1.5), "k": normal(hk), "v": normal(hk),
             "documents": torch.from_numpy(documents).cuda(),
             "prefix": torch.from_numpy(prefix).cuda() if case["prefix"] else None}
    if case["grad"]:
        state["d_o"] = normal(h)
    return state


# ----------------------------------------------------------------- one pass --

def run(state):
    return {"token_logprobs": _run_logprobs, "distillation": _run_distill,
            "span_attention": _run_attention}[state["case"]["op"]](state)


def _own_logprobs(state):
    from torobi_b200 import glue

    case = state["case"]
    if not case["grad"]:
        r = glue.token_logprobs(state["logits"], state["tokens"], top=case["top"],
                                temperature=case["temperature"])
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        if case["top"]:
            out.update(top_logprobs=r.top_logprobs, top_ids=r.top_ids)
        return out
    z = state["logits"].detach().requires_grad_()
    r = glue.token_logprobs(z, state["tokens"], temperature=case["temperature"])
    dz, = torch.autograd.grad((r.logprobs, r.entropy), z,
                              (state["d_logprobs"], state["d_entropy"]))
    return {"logprobs": r.logprobs, "entropy": r.entropy, "d_logits": dz}


def _log_softmax(z, temperature):
    """ln softmax(z / temperature) in 32 bits."""
    x = z.float() / temperature
    x = x - x.amax(1, keepdim=True)
    return x - x.exp().sum(1, keepdim=True).log()


def _top(z, top):
    """The indices of the largest logits, ties to the lowest index: the bits of a float,
    with a negative one's turned over, order as whole numbers; the index breaks ties."""
    bits = (z.float() + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    index = torch.arange(z.shape[1], device=z.device)
    _, ids = (bits * (1 << 31) - index).topk(top, dim=1)
    return ids


def _run_logprobs(state):
    if own:
        return _own_logprobs(state)
    case, z, tokens = state["case"], state["logits"], state["tokens"]
    given = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    logq = _log_softmax(z, case["temperature"])
    q = logq.exp()
    entropy = -torch.where(q > 0, q * logq, 0.0).sum(1)
    out = {"logprobs": torch.where(given, logq.gather(1, at).squeeze(1), 0.0),
           "entropy": entropy}
    if case["top"]:
        out["top_ids"] = _top(z, case["top"])
        out["top_logprobs"] = logq.gather(1, out["top_ids"])
    if case["grad"]:
        g_lp = torch.where(given, state["d_logprobs"], 0.0)
        g_h = state["d_entropy"]
        inner = g_lp[:, None] + g_h[:, None] * (logq + entropy[:, None])
        dz = -torch.where(q > 0, q * inner, 0.0)
        dz.scatter_add_(1, at, g_lp[:, None])
        out["d_logits"] = (dz / case["temperature"]).to(z.dtype)
    return out


def _own_distill(state):
    from torobi_b200 import glue

    case = state["case"]
    targets = state["tokens"] if case["hard"] else None
    z = state["logits"]
    if case["grad"]:
        z = z.detach().requires_grad_()
    r = glue.distillation(z, state["teacher_ids"], state["teacher_logits"], targets=targets,
                          temperature=case["temperature"])
    kl, ce = r if case["hard"] else (r, None)
    out = {"kl": kl}
    if case["hard"]:
        out["ce"] = ce
    if case["grad"]:
        losses, grads = (kl,), (state["d_kl"],)
        if case["hard"]:
            losses, grads = (kl, ce), (state["d_kl"], state["d_ce"])
        out["d_logits"], = torch.autograd.grad(losses, z, grads)
    return out


def _run_distill(state):
    if own:
        return _own_distill(state)
    case, z, tokens = state["case"], state["logits"], state["tokens"]
    temperature = case["temperature"]
    valid = state["teacher_ids"] >= 0
    ids = state["teacher_ids"].long().clamp(min=0)
    t = torch.where(valid, state["teacher_logits"].float() / temperature, float("-inf"))
    t = t - t.amax(1, keepdim=True)
    p = t.exp()
    total = p.sum(1, keepdim=True)
    p = p / total
    logp = t - total.log()
    logq = _log_softmax(z, temperature)
    kl = torch.where(p > 0, p * (logp - logq.gather(1, ids)), 0.0).sum(1)
    out = {"kl": kl}
    given = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    if case["hard"]:
        hard = logq if temperature == 1.0 else _log_softmax(z, 1.0)
        out["ce"] = torch.where(given, -hard.gather(1, at).squeeze(1), 0.0)
    if case["grad"]:
        g_kl = state["d_kl"][:, None] / temperature
        dz = g_kl * logq.exp()
        dz.scatter_add_(1, ids, -g_kl * p)
        if case["hard"]:
            g_ce = torch.where(given, state["d_ce"], 0.0)[:, None]
            dz += g_ce * hard.exp()
            dz.scatter_add_(1, at, -g_ce)
        out["d_logits"] = dz.to(z.dtype)
    return out


def _own_attention(state):
    from torobi_b200 import glue

    first, last = glue.document_spans(state["documents"], state["prefix"])
    if not state["case"]["grad"]:
        o, lse = glue.span_attention_forward(state["q"], state["k"], state["v"], first, last)
        return {"o": o, "lse": lse}
    q, k, v = (state[n].detach().requires_grad_() for n in ("q", "k", "v"))
    o = glue.span_attention(q, k, v, first, last)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), state["d_o"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def _visible(documents, prefix):
    """[batch, query, key]: the key is of the query's document, and not after it or in its
    document's prefix."""
    s = documents.shape[1]
    index = torch.arange(s, device=documents.device)
    new = torch.ones_like(documents, dtype=torch.bool)
    new[:, 1:] = documents[:, 1:] != documents[:, :-1]
    start = torch.where(new, index, 0).cummax(1).values
    until = index + 1 + torch.zeros_like(start)
    if prefix is not None:
        until = torch.maximum(until, start + prefix)
    same = (documents[:, :, None] == documents[:, None, :]) & (documents >= 0)[:, :, None]
    return same & (index < until[:, :, None])


def _run_attention(state):
    if own:
        return _own_attention(state)
    case = state["case"]
    b, s, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    scale = d ** -0.5
    # Query heads of one key/value head side by side: [batch, kv_heads, group, seq, dim].
    q = state["q"].float().view(b, s, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    k = state["k"].float().permute(0, 2, 1, 3)[:, :, None]
    v = state["v"].float().permute(0, 2, 1, 3)[:, :, None]
    see = _visible(state["documents"], state["prefix"])[:, None, None]
    scores = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~see, float("-inf"))
    peak = scores.amax(-1, keepdim=True)
    peak = torch.where(peak == float("-inf"), 0.0, peak)
    p = scores.sub_(peak).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    o = p @ v
    to_rows = lambda x, n: x.permute(0, 3, 1, 2, 4).reshape(b, s, n, d).to(torch.bfloat16)  # noqa: E731
    if not case["grad"]:
        lse = (peak + total.log()).reshape(b, h, s)
        return {"o": to_rows(o, h), "lse": lse}
    d_o = state["d_o"].float().view(b, s, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    dv = (p.transpose(-1, -2) @ d_o).sum(2, keepdim=True)
    dp = d_o @ v.transpose(-1, -2)
    ds = dp.sub_((d_o * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    return {"o": to_rows(o, h), "dq": to_rows(ds @ k, h), "dk": to_rows(dk, hk),
            "dv": to_rows(dv, hk)}


# ------------------------------------------------------------ what it takes --

def work(case):
    if case["op"] == "span_attention":
        pairs = 0
        for length in _lengths(case):
            pre = _prefix_of(case, length)
            pairs += length * (length + 1) // 2 + pre * (pre - 1) // 2
        b, s, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
        flops = 4.0 * b * h * d * pairs
        data = 2 * b * s * d * (2 * h + 2 * hk) + 4 * b * s * (2 if case["prefix"] else 1)
        if case["grad"]:
            return {"bytes": data + 2 * b * s * d * (2 * h + 2 * hk), "flops": 3.5 * flops}
        return {"bytes": data + 4 * b * h * s, "flops": flops}
    n, wide = case["rows"] * case["vocab"], 2 if case["dtype"] == "bf16" else 4
    small = case["rows"] * 8
    if case["op"] == "token_logprobs":
        small += case["rows"] * (8 + 12 * case["top"] + (8 if case["grad"] else 0))
    else:
        small += case["rows"] * case["k"] * (6 if case["compact"] else 12)
    sums = 2 if case["op"] == "distillation" and case["hard"] and case["temperature"] != 1 else 1
    return {"bytes": n * wide * (2 if case["grad"] else 1) + small,
            "flops": n * (6.0 * sums + (6.0 * sums if case["grad"] else 0.0))}


# ------------------------------------------------- the definition in 64 bits --

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "span_attention":
        return _exact_attention(case, state)
    parts = []
    for a in range(0, case["rows"], 256):
        part = {n: x[a:a + 256] if torch.is_tensor(x) else x for n, x in state.items()}
        parts.append(_exact_logprobs(case, part) if case["op"] == "token_logprobs"
                     else _exact_distill(case, part))
    return {n: None if parts[0][n] is None else torch.cat([p[n] for p in parts])
            for n in parts[0]}


def _exact_logprobs(case, state):
    z = state["logits"].double() / case["temperature"]
    lse = z.logsumexp(1)
    q = (z - lse[:, None]).exp()
    # -sum q ln q, as lse - sum q z over what has any probability.
    entropy = lse - (q * torch.where(q > 0, z, 0.0)).sum(1)
    row = torch.arange(len(lse), device=z.device)
    tokens = state["tokens"]
    known = tokens >= 0
    out = {"logprobs": torch.where(known, z[row, tokens] - lse, 0.0), "entropy": entropy}
    if case["top"]:
        out["top_ids"] = None
        out["top_logprobs"] = z.sort(1, descending=True).values[:, :case["top"]] - lse[:, None]
    if case["grad"]:
        a = state["d_logprobs"].double() * known
        c = state["d_entropy"].double()
        hot = torch.zeros_like(z)
        hot[row[known], tokens[known]] = 1.0
        surprise = torch.where(q > 0, z, 0.0) - (lse - entropy)[:, None]
        out["d_logits"] = (a[:, None] * (hot - q) - c[:, None] * q * surprise) / case["temperature"]
    return out


def _exact_distill(case, state):
    heat = case["temperature"]
    z = state["logits"].double()
    ids, rows = state["teacher_ids"].long(), z.shape[0]
    lse = (z / heat).logsumexp(1, keepdim=True)
    teacher = torch.zeros_like(z)
    kl = torch.zeros(rows, dtype=torch.float64, device=z.device)
    weight = (state["teacher_logits"].double() / heat).exp() * (ids >= 0)
    weight = weight / weight.sum(1, keepdim=True)
    for i in range(ids.shape[1]):
        w, at = weight[:, i], ids[:, i].clamp(min=0)
        here = z.gather(1, at[:, None]).squeeze(1) / heat - lse.squeeze(1)
        kl += torch.where(w > 0, w * (w.clamp(min=1e-300).log() - here), 0.0)
        teacher.scatter_add_(1, at[:, None], w[:, None])
    out = {"kl": kl}
    known = state["tokens"] >= 0
    if case["hard"]:
        own_lse = z.logsumexp(1)
        row = torch.arange(rows, device=z.device)
        out["ce"] = torch.where(known, own_lse - z[row, state["tokens"]], 0.0)
    if case["grad"]:
        dz = state["d_kl"].double()[:, None] / heat * ((z / heat - lse).exp() - teacher)
        if case["hard"]:
            hot = torch.zeros_like(z)
            hot[row[known], state["tokens"][known]] = 1.0
            soft = (z - own_lse[:, None]).exp()
            dz += (state["d_ce"].double() * known)[:, None] * (soft - hot)
        out["d_logits"] = dz
    return out


def _exact_attention(case, state):
    """Document by document, with no mask but the order within it."""
    b, s, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    q, k, v = (state[n].double() for n in ("q", "k", "v"))
    o, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    lse = torch.full((b, h, s), float("-inf"), dtype=torch.float64, device=q.device)
    ids = state["documents"].cpu().numpy()
    for row in range(b):
        edges = [0, *(np.flatnonzero(np.diff(ids[row])) + 1).tolist(), s]
        for lo, hi in zip(edges, edges[1:]):
            if ids[row, lo] < 0:
                continue
            n = hi - lo
            pre = int(state["prefix"][row, lo]) if state["prefix"] is not None else 0
            order = torch.arange(n, device=q.device)
            hidden = (order[None, :] > order[:, None]) & (order[None, :] >= pre)
            for g in range(hk):
                heads = range(g * (h // hk), (g + 1) * (h // hk))
                kk, vv = k[row, lo:hi, g], v[row, lo:hi, g]
                for j in heads:
                    x = (q[row, lo:hi, j] @ kk.T) / math.sqrt(d)
                    x = x.masked_fill(hidden, float("-inf"))
                    lse[row, j, lo:hi] = x.logsumexp(1)
                    w = x.softmax(1)
                    o[row, lo:hi, j] = w @ vv
                    if case["grad"]:
                        up = state["d_o"][row, lo:hi, j].double()
                        dw = up @ vv.T
                        dx = w * (dw - (dw * w).sum(1, keepdim=True)) / math.sqrt(d)
                        dq[row, lo:hi, j] = dx @ kk
                        dk[row, lo:hi, g] += dx.T @ q[row, lo:hi, j]
                        dv[row, lo:hi, g] += w.T @ up
    if case["grad"]:
        return {"o": o, "dq": dq, "dk": dk, "dv": dv}
    return {"o": o, "lse": lse}
