"""The answering operators together, as the token loop uses them: adapters on the LM head's logits, the next
id, its log-probability and alternatives, and a prompt's own tokens scored from its hidden rows; through the
engine and its HTTP front end."""
import dataclasses
import http.client
import json
import math
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

# Tolerances. A base logit is the fp32 rounding of a 64-bit sum, off by 2^-24 of its value; an adapter's part
# is off by at most 2e-5 * S, S = scale * sum_j (sum_k |x_k a_jk|) |b_j| (test_gpu_adapters derives it), and the
# sum is rounded once more. So a row's logits are off by e = 2e-5 * max S + 2^-23 * max |l|, the log of
# its sum of exponentials by no more than e, a log-probability by 2 e and the entropy, whose terms move by
# p (2 e) (1 + |log p|), by 4 e per unit of (1 + entropy). The log-probabilities themselves add 1e-4 of
# their value (the head form's bound in test_gpu_logprobs). The synthetic stack has no final norm: logits here
# reach thousands, which is why the bounds go by the rows' own sizes.
REL = 1e-4


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def engine(dev):
    from moe_offload_b200.adapters import AdapterBank
    from moe_offload_b200.engine import OffloadEngine
    from moe_offload_b200.synthetic import C2
    cfg = dataclasses.replace(C2, name="answering_test", layers=3, hidden=512, experts=32, top_k=4, inter=128, seed=7)
    eng = OffloadEngine(budget_pct=50, config=cfg, device=dev, vocab_size=777)
    eng.set_adapters(AdapterBank.synthetic(3, 16, 512, 777, dev, scale=0.2), ["legal", "poetry", "code"])
    yield eng
    eng.close()


def dist(logits):
    """log-softmax of a row in 64 bits."""
    l = logits.astype(np.float64)
    m = l.max()
    return l - m - math.log(np.exp(l - m).sum())


def head_rows(eng, rows, adapter=None):
    """The logits of rows bf16 [T, H] in 64 bits, with an adapter's correction, and how far fp32 ones may be off."""
    x = rows.double()
    out = x @ eng.token_head.head_w.double().t()
    size = torch.zeros_like(out)
    if adapter is not None:
        b = eng.adapters
        low, up, scale = b.a[adapter].double(), b.b[adapter].double(), float(b.scale[adapter])
        out = out + scale * ((x @ low.t()) @ up.t())
        size = abs(scale) * ((x.abs() @ low.abs().t()) @ up.abs().t())
    off = 2e-5 * size.amax(dim=1) + 2.0 ** -23 * out.abs().amax(dim=1)
    return out.cpu().numpy(), off.cpu().numpy()


def check_records(records, ids, rows, n):
    assert [r["id"] for r in records] == list(ids)
    for r, l, e in zip(records, *rows):
        lp = dist(l)
        near = lambda got, want: np.all(np.abs(np.asarray(got) - want) <= 2 * e + REL * np.abs(want) + 1e-12)
        entropy = -float(np.where(lp > -700, np.exp(lp) * lp, 0.0).sum())
        assert near(r["logprob"], lp[r["id"]])
        assert abs(r["entropy"] - entropy) <= 4 * e * (1 + entropy) + REL * entropy + 1e-12
        assert len(r["top"]) == n
        assert near([v for _, v in r["top"]], np.sort(lp)[::-1][:n])
        assert all(near(v, lp[i]) for i, v in r["top"])


@pytest.mark.parametrize("adapter", [None, 0, 2])
def test_prompt_scores(engine, dev, adapter):
    ids = engine.tokenizer.encode("A prompt of some tokens.")
    engine.reset_caches()
    records = engine.score_prompt(ids, 5, adapter=adapter)
    engine.reset_caches()
    rows = engine.stack.prefill(engine.token_head.embed(torch.tensor(ids, dtype=torch.int32, device=dev)))
    check_records(records, ids[1:], head_rows(engine, rows[:-1], adapter), 5)
    assert engine.score_prompt(ids[:1], 3) == []


@pytest.mark.parametrize("temperature", [0.0, 0.9])
@pytest.mark.parametrize("adapter", [None, "poetry"])
def test_generation_with_records(engine, adapter, temperature):
    """Each record belongs to its id, greedy ids head their alternatives, and asking for records or not gives the
    same ids."""
    ids = engine.tokenizer.encode("Once upon")
    scored, prompt = [], []
    engine.reset_caches()
    kw = dict(temperature=temperature, top_p=0.95, seed=3, adapter=adapter)
    got = list(engine.generate_stream(ids, 7, logprobs=4, scored=scored, prompt_scored=prompt, **kw))
    assert [r["id"] for r in scored] == got and [r["id"] for r in prompt] == ids[1:]
    for r in scored:
        assert r["logprob"] <= 0.0 and len(r["top"]) == 4
        if temperature == 0.0:
            assert r["top"][0] == (r["id"], r["logprob"])
        assert sum(math.exp(v) for _, v in r["top"]) <= 1.0 + 1e-5
    engine.reset_caches()
    assert list(engine.generate_stream(ids, 7, **kw)) == got


def test_adapters_change_their_own_generation_only(engine):
    ids = engine.tokenizer.encode("The same prompt")
    runs = {}
    for name in (None, "legal", "code", None):
        engine.reset_caches()
        scored = []
        list(engine.generate_stream(ids, 3, logprobs=1, scored=scored, adapter=name))
        runs.setdefault(name, []).append([r["logprob"] for r in scored])
    assert runs[None][0] == runs[None][1]
    assert runs["legal"][0] != runs[None][0] and runs["code"][0] != runs["legal"][0]


def test_logits_of_four_requests(engine, dev):
    """One decode batch: four rows with their own adapters, or none, then the batch's log-probabilities."""
    from moe_offload_b200.tokens import token_logprobs
    g = torch.Generator(device=dev)
    g.manual_seed(4)
    rows = torch.randn((4, 512), generator=g, device=dev).to(torch.bfloat16)
    of = torch.tensor([2, -1, 0, 2], dtype=torch.int32, device=dev)
    head = engine.token_head
    logits = head.logits(rows, adapters=engine.adapters, adapter_ids=of)
    base = head.logits(rows)
    assert torch.equal(logits[1], base[1]) and not torch.equal(logits[0], base[0])
    ids = head.sample(logits)
    r = token_logprobs(logits, ids, 3)
    for t in range(4):
        assert int(r.top_ids[t, 0]) == int(ids[t])
        record = {"id": int(ids[t]), "logprob": float(r.logprob[t]), "entropy": float(r.entropy[t]),
                  "top": list(zip(r.top_ids[t].tolist(), r.top_logprobs[t].tolist()))}
        check_records([record], [int(ids[t])], head_rows(engine, rows[t:t + 1], None if t == 1 else int(of[t])), 3)


def test_refusals(engine, dev):
    from moe_offload_b200.adapters import AdapterBank
    ids = [1, 2, 3]
    with pytest.raises(ValueError, match="adapter"):
        list(engine.generate_stream(ids, 2, adapter="unknown"))
    with pytest.raises(ValueError, match="adapter"):
        list(engine.generate_stream(ids, 2, adapter=3))
    with pytest.raises(ValueError, match="adapter"):
        engine.score_prompt(ids, adapter=7)
    with pytest.raises(ValueError, match="head"):
        engine.set_adapters(AdapterBank.synthetic(2, 8, 512, 776, dev))
    with pytest.raises(ValueError, match="name"):
        engine.set_adapters(engine.adapters, ["a", "a", "b"])
    assert engine.adapter_names == ["legal", "poetry", "code"]


def test_over_http(engine):
    from moe_offload_b200.server import make_server
    srv = make_server(engine, "127.0.0.1", 0, model_id="base")
    threading.Thread(target=srv.serve_forever, daemon=True).start()
    try:
        c = http.client.HTTPConnection("127.0.0.1", srv.server_address[1], timeout=60)
        c.request("POST", "/v1/completions", body=json.dumps({"prompt": "Hello", "max_tokens": 3, "logprobs": 5, "echo": True,
                                                               "model": "code"}))
        out = json.loads(c.getresponse().read())
        c.close()
        lp = out["choices"][0]["logprobs"]
        assert out["model"] == "code" and lp["tokens"][:5] == list("Hello")
        assert lp["token_logprobs"][0] is None and all(v <= 0 for v in lp["token_logprobs"][1:])
        assert all(len(t) == 5 for t in lp["top_logprobs"][1:])
    finally:
        srv.shutdown()
        srv.server_close()
