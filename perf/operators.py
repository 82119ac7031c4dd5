"""Cases of the answering side of the token loop: low-rank adapters of many requests beside a
shared projection, log-probabilities (with entropy and the top alternatives) of logits that
are in memory, and the same straight from hidden rows and the LM head.

    adapters   y + scale[a] * (x . A[a]^T) . B[a]^T for rows x [T, K], y [T, N], a = ids[t];
               a row with id -1 keeps y. y is bf16 (a hidden projection) or fp32 (logits).
    logprobs   fp32 logits [T, V], target ids [T] (-1: none, NaN) -> log-probability of the
               target, entropy in nats, the n largest logits' ids (ties: the lowest id first)
               and their log-probabilities.
    score      the same from bf16 rows [T, H] and the bf16 head [V, H]. A logit is the fp32
               rounding of the products' sum in 64 bits, as everywhere in the token loop, and
               ids are ordered by it.

Sizes: hidden 2,048 / 3,072, inner 768 and vocabulary 248,320 are the decode configurations';
the others are generic."""
import math

import torch

own = False


def listed():
    return [
        # one decode step of one request, with 20 alternatives of the full vocabulary
        {"name": "logprobs_step", "op": "logprobs", "T": 1, "V": 248320, "n": 20, "masked": 0.0},
        # four rows of a byte-sized vocabulary: launch latency alone
        {"name": "logprobs_bytes", "op": "logprobs", "T": 4, "V": 257, "n": 5, "masked": 0.0},
        # a decode batch under a grammar mask that leaves a tenth of an odd vocabulary
        {"name": "logprobs_batch_masked", "op": "logprobs", "T": 64, "V": 50021, "n": 5, "masked": 0.9},
        # the logits of a 512-row chunk of prompt
        {"name": "logprobs_chunk", "op": "logprobs", "T": 512, "V": 248320, "n": 20, "masked": 0.0},
        # scoring the one row behind a decode step
        {"name": "score_step", "op": "score", "T": 1, "V": 248320, "H": 3072, "n": 5},
        # a short odd prompt on a smaller head
        {"name": "score_short", "op": "score", "T": 33, "V": 32003, "H": 2048, "n": 0},
        # a prompt of ordinary length
        {"name": "score_prompt", "op": "score", "T": 256, "V": 248320, "H": 3072, "n": 5},
        # the prefill configuration's prompt, all alternatives
        {"name": "score_prefill", "op": "score", "T": 2048, "V": 248320, "H": 3072, "n": 20},
        # one token of one request through one projection
        {"name": "adapters_step", "op": "adapters", "T": 1, "K": 2048, "N": 768, "r": 8, "banks": 4, "mix": "one", "y": "bf16"},
        # a decode batch in which nearly each row has an adapter of its own
        {"name": "adapters_batch", "op": "adapters", "T": 64, "K": 3072, "N": 768, "r": 16, "banks": 48, "mix": "rows", "y": "bf16"},
        # adapters on the LM head, beside fp32 logits of four requests
        {"name": "adapters_head", "op": "adapters", "T": 4, "K": 3072, "N": 248320, "r": 16, "banks": 8, "mix": "rows", "y": "f32"},
        # a prefill batch of several requests, the rows of each together, some without an adapter
        {"name": "adapters_prefill", "op": "adapters", "T": 2048, "K": 768, "N": 3072, "r": 64, "banks": 6, "mix": "runs", "y": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "score", "adapters"])
    if op == "logprobs":
        V = _log(rng, 257, 248320)
        return {"op": op, "T": min(_log(rng, 1, 2048), 512 * 248320 // V), "V": V, "n": rng.randint(0, min(20, V)),
                "masked": rng.choice([0.0, 0.0, 0.5, 0.99])}
    if op == "score":
        return {"op": op, "T": _log(rng, 1, 2048), "V": _log(rng, 257, 248320), "H": 8 * _log(rng, 32, 384),
                "n": rng.randint(0, 20)}
    y = rng.choice(["bf16", "bf16", "f32"])
    T = _log(rng, 1, 2048)
    N = _log(rng, 64, 4096) if y == "bf16" else min(_log(rng, 257, 248320), max(257, (1 << 22) // T))
    return {"op": op, "T": T, "K": 8 * _log(rng, 32, 384), "N": N, "r": rng.choice([8, 16, 24, 32, 64, 128]),
            "banks": rng.randint(1, 64), "mix": rng.choice(["one", "rows", "runs"]), "y": y}


def _ids(case, g):
    """The adapter of each row: one for all; each row its own choice; or runs of rows of a request."""
    T, n = case["T"], case["banks"]
    dev = g.device
    if case["mix"] == "one":
        return torch.randint(0, n, (1,), generator=g, device=dev, dtype=torch.int32).expand(T).contiguous()
    if case["mix"] == "rows":
        return torch.randint(-1, n, (T,), generator=g, device=dev, dtype=torch.int32)
    runs = 8
    of = torch.randint(-1, n, (runs,), generator=g, device=dev, dtype=torch.int32)
    cut = torch.randint(0, T + 1, (runs - 1,), generator=g, device=dev).sort().values
    return of[torch.searchsorted(cut, torch.arange(T, device=dev), right=True)]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)

    op, T = case["op"], case["T"]
    if op == "adapters":
        K, N, r, n = case["K"], case["N"], case["r"], case["banks"]
        return {"op": op, "x": normal(T, K), "y": normal(T, N, dtype=torch.bfloat16 if case["y"] == "bf16" else torch.float32),
                "a": normal(n, r, K, std=K ** -0.5), "b": normal(n, N, r, std=r ** -0.5),
                "scale": torch.rand((n,), generator=g, device=dev) + 0.5, "ids": _ids(case, g)}
    V = case["V"]
    targets = torch.randint(0, V, (T,), generator=g, device=dev, dtype=torch.int32)
    if T > 1:
        targets[-1] = -1                                     # the last row of a prompt has no next token
    if op == "score":
        head, h = normal(V, case["H"], std=0.02), normal(T, case["H"])
        # rows whose next token the model expects: the hidden row leans towards that token's head row
        lean = torch.rand((T, 1), generator=g, device=dev).square() * 25.0
        h = (h + lean * head[targets.clamp(min=0).long()].float()).to(torch.bfloat16)
        return {"op": op, "head": head, "h": h, "targets": targets, "n": case["n"]}
    logits = normal(T, V, std=3.0, dtype=torch.float32)
    lean = torch.rand((T,), generator=g, device=dev).square() * 40.0
    logits[torch.arange(T, device=dev), targets.clamp(min=0).long()] += lean
    if case["masked"]:
        gone = torch.rand((T, V), generator=g, device=dev) < case["masked"]
        gone[torch.arange(T, device=dev), targets.clamp(min=0).long()] = False
        logits.masked_fill_(gone, -math.inf)
    return {"op": op, "logits": logits, "targets": targets, "n": case["n"]}


def _order(x):
    """int64 keys whose order is that of the fp32 values, equal ones the lowest column first."""
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, (-(1 << 31)) - bits - 1, bits)
    return bits * (1 << 32) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))


def _plain_logprobs(logits, targets, n):
    """logits fp32 [T, V]; statistics in 64 bits, for the rows whose probability is all but one."""
    top = torch.topk(_order(logits), n, dim=1).indices
    z = logits.double()
    z = z - z.amax(dim=1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(dim=1, keepdim=True)
    lse = torch.log(total)
    entropy = lse[:, 0] - torch.where(e > 0, e * z, 0.0).sum(dim=1) / total[:, 0]
    at = targets.long()
    lp = torch.where(at >= 0, torch.gather(z, 1, at.clamp(min=0)[:, None])[:, 0] - lse[:, 0], math.nan)
    return {"logprob": lp.float(), "entropy": entropy.float(), "top_ids": top.int(),
            "top_logprobs": (torch.gather(z, 1, top) - lse).float()}


def run(state):
    op = state["op"]
    if own:
        if op == "adapters":
            from moe_offload_b200.adapters import AdapterBank
            return AdapterBank(state["a"], state["b"], state["scale"]).add(state["y"], state["x"], state["ids"])
        from moe_offload_b200 import tokens
        if op == "logprobs":
            r = tokens.token_logprobs(state["logits"], state["targets"], state["n"])
        else:
            r = tokens.head_logprobs(state["head"], state["h"], state["targets"], state["n"])
        return {"logprob": r.logprob, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    if op == "adapters":
        at = state["ids"].long()
        a, b = state["a"][at.clamp(min=0)].float(), state["b"][at.clamp(min=0)].float()
        u = torch.bmm(a, state["x"].float()[:, :, None])
        delta = torch.bmm(b, u)[:, :, 0] * state["scale"][at.clamp(min=0)][:, None]
        y = state["y"]
        return torch.where((at >= 0)[:, None], (y.float() + delta).to(y.dtype), y)
    if op == "logprobs":
        return _plain_logprobs(state["logits"], state["targets"], state["n"])
    # 64 bits: the order of the alternatives is that of logits rounded once to fp32
    logits = torch.matmul(state["h"].double(), state["head"].double().t()).float()
    return _plain_logprobs(logits, state["targets"], state["n"])


def _distinct(case):
    """How many adapters a case's rows are expected to use."""
    n, T = case["banks"], case["T"]
    if case["mix"] == "one":
        return 1.0
    picks = T if case["mix"] == "rows" else min(T, 8)
    return n * (1.0 - (1.0 - 1.0 / (n + 1)) ** picks)


def work(case):
    T = case["T"]
    if case["op"] == "adapters":
        K, N, r = case["K"], case["N"], case["r"]
        ysize = 2 if case["y"] == "bf16" else 4
        return {"bytes": 2.0 * T * K + 2.0 * ysize * T * N + 2.0 * r * (K + N) * _distinct(case) + 4 * T,
                "flops": 2.0 * T * r * (K + N)}
    out = T * (12 + 8 * case["n"])
    if case["op"] == "logprobs":
        return {"bytes": 4.0 * T * case["V"] + out, "flops": 5.0 * T * case["V"]}
    return {"bytes": 2.0 * case["H"] * (case["V"] + T) + out, "flops": 2.0 * T * case["V"] * case["H"]}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "adapters":
        out = s["y"].double()
        for k in range(case["banks"]):
            rows = (s["ids"] == k).nonzero()[:, 0]
            if rows.numel():
                low = s["x"][rows].double() @ s["a"][k].double().t()
                out[rows] += s["scale"][k].double() * (low @ s["b"][k].double().t())
        return out
    got = {"logprob": [], "entropy": [], "top_logprobs": []}
    rows = s["h"] if s["op"] == "score" else s["logits"]
    for i in range(0, case["T"], 256):
        logits = rows[i:i + 256].double()
        if s["op"] == "score":
            logits = logits @ s["head"].double().t()
        lp = logits - torch.logsumexp(logits, dim=1, keepdim=True)
        at = s["targets"][i:i + 256].long()
        picked = lp[torch.arange(at.numel(), device=lp.device), at]
        got["logprob"].append(torch.where(at < 0, torch.full_like(picked, math.nan), picked))
        got["entropy"].append(torch.special.entr(lp.exp()).sum(dim=1))
        got["top_logprobs"].append(lp.sort(dim=1, descending=True).values[:, :case["n"]] if case["n"] else lp[:, :0])
    return {**{k: torch.cat(v) for k, v in got.items()}, "top_ids": None}
