"""What a request of a shared batch brings of its own, measured operator by operator: the rules its tokens are drawn
under, the log-probabilities it asks for, and its low-rank adapter beside the weights that all requests share.

A case is one of

* ``op="sample"``: ``rows`` rows of ``vocab`` float32 logits, each with a temperature, a top-k, a top-p and a min-p of its
  own, drawn as ``rule`` says (``k``, ``p``, ``m``: the filters in use; ``mixed``: rows of every kind, greedy ones among
  them), and a given uniform number;
* ``op="logprobs"``: ``rows`` rows of ``vocab`` logits and a token of each;
* ``op="lora"``: rows of ``k`` numbers times the adapters of their requests, added to ``into`` (rows of ``n`` numbers, in
  the activation type, or in 32 bits where they are the residual stream).  ``decoding`` rows are requests of their own, each
  with an adapter; ``portions`` are the lengths of prompts that run beside them.  ``count`` adapters of rank ``rank`` are
  loaded; a site of ``parts`` projections (q, k and v; gate and up) has that many inner products, whose columns are
  ``n`` split at ``cuts``.
"""

from __future__ import annotations

import math

import torch

own = False

VOCAB_SMALL, VOCAB_LARGE = 151936, 152064  # of the 0.5B and 3B shapes, and of the larger ones

# what a layer's four products look like: (k, columns of each projection that reads the rows, residual stream behind it)
SITES = {
    "0.5b-qkv": (896, (896, 128, 128), False), "0.5b-o": (896, (896,), True),
    "0.5b-gate-up": (896, (4864, 4864), False), "0.5b-down": (4864, (896,), True),
    "3b-qkv": (2048, (2048, 256, 256), False), "3b-o": (2048, (2048,), True),
    "3b-gate-up": (2048, (11008, 11008), False), "3b-down": (11008, (2048,), True),
    "7b-qkv": (3584, (3584, 512, 512), False), "7b-o": (3584, (3584,), True),
    "7b-gate-up": (3584, (18944, 18944), False), "7b-down": (18944, (3584,), True),
}


def _sample(rows, vocab, rule, name=None):
    case = dict(op="sample", rows=rows, vocab=vocab, rule=rule)
    return dict(case, name=name) if name else case


def _logprobs(rows, vocab, name=None):
    case = dict(op="logprobs", rows=rows, vocab=vocab)
    return dict(case, name=name) if name else case


def _lora(site, rank, count, decoding=0, portions="", dtype="bfloat16", name=None):
    case = dict(op="lora", site=site, rank=rank, count=count, decoding=decoding, portions=portions, dtype=dtype)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one user's chat under the usual rules: launches and latency only
        _sample(1, VOCAB_SMALL, "kp", "sample-1-kp"),
        # the benchmark's eight sequences, nucleus sampling alone
        _sample(8, VOCAB_SMALL, "p", "sample-8-p"),
        # a busy server, where every request has rules of its own
        _sample(64, VOCAB_SMALL, "mixed", "sample-64-mixed"),
        # many samples of few prompts, as data for training is generated
        _sample(256, VOCAB_LARGE, "kpm", "sample-256-kpm"),
        # the drawn tokens' log-probabilities in a decode step
        _logprobs(8, VOCAB_SMALL, "logprobs-8"),
        # a prompt is scored: every position of a full step
        _logprobs(2048, VOCAB_SMALL, "logprobs-2048"),
        # one request with an adapter: launches and latency only
        _lora("3b-qkv", 16, 4, decoding=1, name="lora-qkv-1"),
        # a busy server: 64 requests on 16 adapters, the widest product of a layer
        _lora("3b-gate-up", 16, 16, decoding=64, name="lora-gate-up-64"),
        # ... and the one with the longest sums, into the residual stream
        _lora("7b-down", 32, 8, decoding=24, name="lora-down-24"),
        # short questions that arrive together beside decoding requests, each tenant with an adapter
        _lora("3b-qkv", 16, 8, decoding=5, portions="37,311,129,64,72", name="lora-qkv-ragged"),
        # two long prompts of large adapters fill a step
        _lora("7b-gate-up", 64, 4, portions="1271,777", name="lora-gate-up-2048"),
        # the 32-bit path over a prompt
        _lora("3b-o", 8, 3, decoding=3, portions="517", dtype="float32", name="lora-o-fp32"),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("sample", "sample", "logprobs", "lora", "lora", "lora"))
    vocab = rng.choice((VOCAB_SMALL, VOCAB_LARGE, rng.randint(20000, 150000)))
    if op == "sample":
        return _sample(_log(rng, 1, 200), vocab, rng.choice(("k", "p", "m", "kp", "pm", "kpm", "mixed")))
    if op == "logprobs":
        return _logprobs(_log(rng, 1, 1500), vocab)
    site = rng.choice([s for s in SITES if s != "7b-gate-up"])
    dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
    rank = rng.choice((4, 8, 12, 16, 24, 32, 64))
    decoding = _log(rng, 1, 64)
    portions = [_log(rng, 2, 600) for _ in range(rng.choice((0, 0, 1, 3)))]
    return _lora(site, rank, _log(rng, 1, 16), decoding, ",".join(map(str, portions)), dtype)


# ---------------------------------------------------------------- inputs
def _logits(rows, vocab, g):
    """Rows as a trained model leaves them: a broad bulk, and some dozens of tokens that stand out of it."""
    spread = torch.rand(rows, 1, generator=g, device="cuda") * 1.5 + 1.5
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * spread
    likely = torch.randint(vocab, (rows, 64), generator=g, device="cuda")
    lift = -torch.log(torch.rand(rows, 64, generator=g, device="cuda") + 1e-6) * 1.5 + 7.0
    return logits.scatter_add_(1, likely, lift)


def _rules(rows, rule, g):
    pick = lambda values: torch.tensor(values, device="cuda")[  # noqa: E731
        torch.randint(len(values), (rows,), generator=g, device="cuda")]
    temperature = pick([0.0, 0.6, 0.8, 1.0, 1.3] if rule == "mixed" else [0.6, 0.8, 1.0, 1.0, 1.2])
    top_k, top_p, min_p = pick([10, 20, 40, 50, 100, 1000]), pick([0.5, 0.8, 0.9, 0.95, 0.99]), pick([0.01, 0.02, 0.05, 0.1])
    if rule == "mixed":  # every filter off in half of the rows
        on = torch.rand(3, rows, generator=g, device="cuda") < 0.5
    else:
        on = torch.tensor([[letter in rule] for letter in "kpm"], device="cuda").expand(3, rows)
    return {"temperature": temperature, "top_k": torch.where(on[0], top_k, 0).to(torch.int32),
            "top_p": torch.where(on[1], top_p, 1.0), "min_p": torch.where(on[2], min_p, 0.0)}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    if case["op"] != "lora":
        rows, vocab = case["rows"], case["vocab"]
        state = {"op": case["op"], "logits": _logits(rows, vocab, g)}
        if case["op"] == "sample":
            state.update(_rules(rows, case["rule"], g))
            # uniform numbers of 24 bits, as the framework makes them
            state["uniform"] = torch.randint(1 << 24, (rows,), generator=g, device="cuda").float() / (1 << 24)
        else:
            state["tokens"] = torch.randint(vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        return state
    k, columns, stream = SITES[case["site"]]
    dtype = getattr(torch, case["dtype"])
    count, rank, parts, n = case["count"], case["rank"], len(columns), sum(columns)
    lengths = [1] * case["decoding"] + [int(p) for p in case["portions"].split(",") if p]
    # a request's adapter; one request in nine has none
    chosen = torch.randint(9 * count, (len(lengths),), generator=g, device="cuda")
    chosen = torch.where(chosen < count, -1, chosen % count).to(torch.int32)
    adapters = torch.repeat_interleave(chosen, torch.tensor(lengths, device="cuda"))
    rows = sum(lengths)
    draw_ = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    return {
        "op": "lora", "x": draw_(rows, k).to(dtype), "down": (draw_(count, parts * rank, k) * k ** -0.5).to(dtype),
        "up": (draw_(count, n, rank) * rank ** -0.5 * 0.25).to(dtype),
        "scale": 0.5 + 1.5 * torch.rand(count, generator=g, device="cuda"), "adapters": adapters, "columns": columns,
        "into": draw_(rows, n).to(torch.float32 if stream else dtype),
        "part_of_column": torch.repeat_interleave(torch.arange(parts, device="cuda"), torch.tensor(columns, device="cuda")),
    }


# ---------------------------------------------------------------- one pass
def _plain_sample(s):
    # 64 bits: which token a running sum passes a share of the whole at, and where a share of the weight ends
    values, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    vocab = values.shape[1]
    column = lambda name: s[name].double()[:, None]  # noqa: E731
    temperature = column("temperature")
    safe = torch.where(temperature > 0, temperature, 1.0)
    weight = torch.exp((values.double() - values[:, :1].double()) / safe)
    least = weight >= column("min_p")
    top_k = s["top_k"][:, None]
    rank = torch.arange(vocab, device=values.device)[None, :]
    weight = weight * ((top_k <= 0) | (rank < top_k))
    before = torch.cumsum(weight, 1) - weight
    top_p = column("top_p")
    total = weight.sum(1, keepdim=True)
    weight = weight * ((top_p >= 1) | (before < top_p * total) | (rank == 0)) * least
    kept = torch.zeros_like(weight).scatter_(1, order, weight)
    running = torch.cumsum(kept, 1)
    passed = (running <= column("uniform") * running[:, -1:]).sum(1)
    # (rounding may leave the last token with any weight unpassed)
    last = (running < running[:, -1:]).sum(1)
    drawn = torch.minimum(passed, last)
    return torch.where(s["temperature"] > 0, drawn, order[:, 0]).to(torch.int32)


def _plain_logprobs(s):
    logits = s["logits"]
    best = logits.amax(1, keepdim=True)
    total = torch.exp(logits - best).sum(1)
    return (logits.gather(1, s["tokens"].long()[:, None])[:, 0] - best[:, 0]) - torch.log(total)


def _plain_lora(s):
    # all adapters over all rows; what is not a row's own counts nothing
    x, down, up, adapters = s["x"].float(), s["down"].float(), s["up"].float(), s["adapters"]
    count, inner, k = down.shape
    n, rank = up.shape[1:]
    parts = inner // rank
    mine = (adapters[:, None] == torch.arange(count, device=x.device)[None, :]) * s["scale"][None, :]
    hidden = (x @ down.reshape(count * inner, k).t()).reshape(-1, count, inner) * mine[:, :, None]
    reads = (s["part_of_column"][:, None] == torch.arange(parts, device=x.device)[None, :]).float()
    wide = up.permute(1, 0, 2)[:, :, None, :] * reads[:, None, :, None]  # [n, count, parts, rank]
    out = s["into"].float() + hidden.reshape(-1, count * inner) @ wide.reshape(n, count * inner).t()
    return out.to(s["into"].dtype)


def run(state):
    if own:
        from cie_amd.kernels import ops

        if state["op"] == "sample":
            return ops.sample(state["logits"], state["temperature"], state["uniform"], top_k=state["top_k"],
                              top_p=state["top_p"], min_p=state["min_p"])
        if state["op"] == "logprobs":
            return ops.token_logprobs(state["logits"], state["tokens"])
        return ops.lora_add(state["x"], state["down"], state["up"], state["scale"], state["adapters"], state["into"],
                            columns=state["columns"], out=torch.empty_like(state["into"]))
    return {"sample": _plain_sample, "logprobs": _plain_logprobs, "lora": _plain_lora}[state["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] != "lora":
        rows, vocab = case["rows"], case["vocab"]
        given = 5 if case["op"] == "sample" else 1  # numbers a row brings beside its logits
        return {"bytes": 4 * rows * (vocab + given + 1), "flops": 4 * rows * vocab}
    k, columns, stream = SITES[case["site"]]
    size = 2 if case["dtype"] == "bfloat16" else 4
    n, parts, rank = sum(columns), len(columns), case["rank"]
    lengths = [1] * case["decoding"] + [int(p) for p in case["portions"].split(",") if p]
    rows, used = sum(lengths), min(case["count"], len(lengths))
    read = rows * k * size + used * rank * (parts * k + n) * size + rows * 4 + case["count"] * 4
    return {"bytes": read + 2 * rows * n * (4 if stream else size), "flops": 2 * rows * rank * (parts * k + n)}


# ---------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    import numpy as np

    state = prepare(case, seed)
    if case["op"] == "sample":
        if case["rows"] > 300:
            return None
        logits = state["logits"].cpu().numpy()
        rules = {name: state[name].cpu().numpy().astype(np.float64) for name in
                 ("temperature", "top_k", "top_p", "min_p", "uniform")}
        tokens = []
        for r, row in enumerate(logits.astype(np.float64)):
            t, k, p, m, u = (rules[name][r] for name in ("temperature", "top_k", "top_p", "min_p", "uniform"))
            if not t > 0:
                tokens.append(int(row.argmax()))
                continue
            order = np.argsort(-row, kind="stable")
            if 0 < k < len(row):
                order = order[: int(k)]
            weights = np.exp((row[order] - row[order[0]]) / t)
            if p < 1:
                share = np.cumsum(weights)
                order = order[: max(1, int(np.searchsorted(share, p * share[-1], side="left")) + 1)]
                weights = weights[: len(order)]
            order = order[weights >= m]
            chosen = np.sort(order)
            running = np.cumsum(np.exp((row[chosen] - row.max()) / t))
            place = int(np.searchsorted(running, u * running[-1], side="right"))
            tokens.append(int(chosen[min(place, len(chosen) - 1)]))
        return torch.tensor(tokens, dtype=torch.int32)
    if case["op"] == "logprobs":
        out = []
        for rows, tokens in zip(state["logits"].split(128), state["tokens"].split(128)):
            wide = rows.double()
            out.append(wide[torch.arange(len(rows), device=wide.device), tokens.long()] - torch.logsumexp(wide, 1))
        return torch.cat(out)
    out = state["into"].double()
    rank = case["rank"]
    for a in range(case["count"]):
        rows = (state["adapters"] == a).nonzero()[:, 0]
        inner = state["x"][rows].double() @ state["down"][a].double().t()
        begin = 0
        for part, width in enumerate(state["columns"]):
            factor = state["up"][a, begin: begin + width].double()
            out[rows, begin: begin + width] += float(state["scale"][a]) * (inner[:, part * rank: (part + 1) * rank] @ factor.t())
            begin += width
    return out
