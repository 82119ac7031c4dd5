"""Host side of log-probabilities and adapters, without a GPU: refusals of the C entry points (checked
before any CUDA call) and of the Python wrappers, the OpenAI response shapes of `logprobs` and `echo`,
and adapters chosen by model name, over a stand-in engine."""
import http.client
import json
import threading

import pytest
import torch


@pytest.fixture(scope="module")
def call():
    from moe_offload_b200 import _lib
    return _lib.call


def refused(call, name, *args, what=""):
    from moe_offload_b200._lib import MoeError
    with pytest.raises(MoeError) as e:
        call(name, *args)
    assert e.value.rc == -22 and what in str(e.value), str(e.value)


def test_token_logprobs_refusals(call):
    f, p = "moe_token_logprobs", 4096                                # (addresses that are never read)
    refused(call, f, p, 0, 10, None, 0, None, p, None, None, None, what="T=0")
    refused(call, f, p, 1, 0, None, 0, None, p, None, None, None, what="V=0")
    refused(call, f, p, 1, (1 << 30) + 1, None, 0, None, p, None, None, None, what="V")
    refused(call, f, p, 1, 100, None, 33, None, p, p, p, None, what="n=33")
    refused(call, f, p, 1, 100, None, -1, None, p, p, p, None, what="n=-1")
    refused(call, f, p, 1, 5, None, 6, None, p, p, p, None, what="n=6")
    refused(call, f, p, 1, 100, None, 3, None, p, None, p, None, what="null")
    refused(call, f, p, 1, 100, None, 3, None, p, p, None, None, what="null")
    refused(call, f, p, 1, 100, p, 0, None, p, None, None, None, what="null")
    refused(call, f, p, 1, 100, None, 0, p, p, None, None, None, what="null")
    refused(call, f, p, 1, 100, None, 0, None, None, None, None, None, what="null")
    refused(call, f, None, 1, 100, None, 0, None, p, None, None, None, what="logits")
    refused(call, f, p + 2, 1, 100, None, 0, None, p, None, None, None, what="aligned")


def test_head_logprobs_refusals(call):
    f, p = "moe_head_logprobs", 4096
    tail = (None, 0, None, p, None, None, p, 1 << 40, None)
    refused(call, f, p, 0, 64, p, 1, *tail, what="V=0")
    refused(call, f, p, 100, 64, p, 0, *tail, what="T=0")
    refused(call, f, p, 100, 60, p, 1, *tail, what="H=60")
    refused(call, f, p, 100, 8200, p, 1, *tail, what="H=8200")
    refused(call, f, None, 100, 64, p, 1, *tail, what="head")
    refused(call, f, p, 100, 64, None, 1, *tail, what="x")
    refused(call, f, p + 8, 100, 64, p, 1, *tail, what="16-byte")
    refused(call, f, p, 100, 64, p + 2, 1, *tail, what="16-byte")
    refused(call, f, p, 100, 64, p, 1, None, 40, None, p, p, p, p, 1 << 40, None, what="n=40")


def test_adapter_add_refusals(call):
    f = "moe_adapter_add"
    x, a, b, s, ids, y, out = (k << 24 for k in range(1, 8))         # far apart, never read

    def args(T=4, K=64, N=64, ad=2, r=8, x=x, a=a, b=b, s=s, ids=ids, y=y, fp32=0, out=out):
        return (x, T, K, N, a, b, s, ad, r, ids, y, fp32, out, None)
    for bad, what in ((dict(T=0), "T=0"), (dict(K=60), "K=60"), (dict(K=0), "K=0"), (dict(N=0), "N=0"),
                      (dict(ad=0), "adapters=0"), (dict(r=0), "rank=0"), (dict(r=12), "rank=12"), (dict(r=136), "rank=136"),
                      (dict(x=None), "null"), (dict(ids=None), "null"), (dict(out=None), "null"),
                      (dict(x=x + 8), "16-byte"), (dict(a=a + 2), "16-byte"), (dict(b=b + 8), "16-byte"),
                      (dict(y=y + 1), "aligned"), (dict(out=out + 2, fp32=1), "aligned"),
                      (dict(out=y + 64), "overlap"), (dict(out=x), "overlap"), (dict(out=a + 512), "overlap"),
                      (dict(out=b), "overlap"), (dict(out=s, N=8), "overlap"), (dict(out=ids), "overlap")):
        refused(call, f, *args(**bad), what=what)


def test_wrappers_refuse_host_tensors():
    from moe_offload_b200.adapters import AdapterBank
    from moe_offload_b200.tokens import head_logprobs, token_logprobs
    bf = torch.bfloat16
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        head_logprobs(torch.zeros(8, 8, dtype=bf), torch.zeros(2, 8, dtype=bf))
    with pytest.raises(ValueError, match="CUDA"):
        AdapterBank(torch.zeros(1, 8, 8, dtype=bf), torch.zeros(1, 8, 8, dtype=bf), torch.ones(1))


# ------------------------------------------------------------------ the server over a stand-in engine

REPLY = "Hi! \xe9 ok"


class Engine:
    adapter_names = ["legal", "poetry"]

    def __init__(self):
        from moe_offload_b200.tokens import ByteTokenizer
        self.tokenizer = ByteTokenizer(300)
        self.calls = []
        self._last_timings = {}

    @staticmethod
    def record(i, n):
        return {"id": i, "logprob": -0.25 * (i % 4), "entropy": 1.0,
                "top": [((i + k) % 300, float("-inf") if k == 2 else -0.25 * k) for k in range(n)]}

    def generate_stream(self, prompt_ids, max_tokens, temperature=0.0, top_p=1.0, stop_ids=None, seed=0, adapter=None,
                        logprobs=None, scored=None, prompt_scored=None):
        self.calls.append(dict(adapter=adapter, logprobs=logprobs, echo=prompt_scored is not None))
        if prompt_scored is not None:
            prompt_scored += [self.record(i, logprobs) for i in prompt_ids[1:]]
        for i in self.tokenizer.encode(REPLY)[:max_tokens]:
            if logprobs is not None:
                scored.append(self.record(i, logprobs))
            yield i

    def _snapshot_decode_totals(self):
        return (0, 0, 0, 0, 0, 0)


@pytest.fixture()
def server():
    from moe_offload_b200.server import make_server
    eng = Engine()
    srv = make_server(eng, "127.0.0.1", 0, model_id="base", default_max_tokens=64)
    threading.Thread(target=srv.serve_forever, daemon=True).start()
    yield srv, eng
    srv.shutdown()
    srv.server_close()


def post(srv, path, body):
    c = http.client.HTTPConnection("127.0.0.1", srv.server_address[1], timeout=10)
    c.request("POST", path, body=json.dumps(body), headers={"Content-Type": "application/json"})
    r = c.getresponse()
    data = r.read()
    c.close()
    return r.status, data


def strict(data):
    return json.loads(data, parse_constant=lambda c: pytest.fail(f"{c} is no JSON"))


def test_completion_logprobs(server):
    srv, eng = server
    st, data = post(srv, "/v1/completions", {"prompt": "abc", "max_tokens": 6, "logprobs": 3})
    assert st == 200
    choice = strict(data)["choices"][0]
    ids = REPLY.encode()[:6]
    lp = choice["logprobs"]
    assert lp["tokens"] == ["H", "i", "!", " ", "token_id:195", "token_id:169"]
    assert lp["token_logprobs"] == [-0.25 * (i % 4) for i in ids]
    assert lp["top_logprobs"][0] == {"H": 0.0, "I": -0.25, "J": None}
    assert lp["text_offset"][:5] == [0, 1, 2, 3, 4]
    st, data = post(srv, "/v1/completions", {"prompt": "abc", "max_tokens": 2})
    assert "logprobs" not in strict(data)["choices"][0]
    assert [c["logprobs"] for c in eng.calls] == [3, None]


def test_completion_echo(server):
    srv, eng = server
    st, data = post(srv, "/v1/completions", {"prompt": "abc", "max_tokens": 2, "logprobs": 1, "echo": True})
    choice = strict(data)["choices"][0]
    assert choice["text"] == "abcHi"
    lp = choice["logprobs"]
    assert lp["tokens"] == ["a", "b", "c", "H", "i"] and lp["text_offset"] == [0, 1, 2, 3, 4]
    assert lp["token_logprobs"][0] is None and lp["top_logprobs"][0] is None
    assert lp["token_logprobs"][1:] == [-0.25 * (i % 4) for i in b"bcHi"]
    assert eng.calls[-1]["echo"]
    st, data = post(srv, "/v1/completions", {"prompt": "abc", "max_tokens": 2, "echo": True})
    assert strict(data)["choices"][0] == {"index": 0, "text": "abcHi", "finish_reason": "length"}


def test_chat_logprobs_and_stream(server):
    srv, _ = server
    body = {"messages": [{"role": "user", "content": "x"}], "max_tokens": 30, "logprobs": True, "top_logprobs": 2}
    st, data = post(srv, "/v1/chat/completions", body)
    content = strict(data)["choices"][0]["logprobs"]["content"]
    assert [c["token"] for c in content][:3] == ["H", "i", "!"]
    assert content[0]["bytes"] == [72] and [t["token"] for t in content[0]["top_logprobs"]] == ["H", "I"]
    for path, req in (("/v1/chat/completions", body),
                      ("/v1/completions", {"prompt": "ab", "max_tokens": 30, "logprobs": 0, "echo": True})):
        st, data = post(srv, path, {**req, "stream": True})
        events = [strict(e[6:]) for e in data.decode().split("\n\n") if e.startswith("data: {")]
        choices = [e["choices"][0] for e in events]
        if path.endswith("chat/completions"):
            text = "".join(c["delta"].get("content", "") for c in choices)
            tokens = [t["token"] for c in choices for t in c.get("logprobs", {}).get("content", [])]
            assert text == REPLY and len(tokens) == len(REPLY.encode())
        else:
            text = "".join(c["text"] for c in choices)
            tokens = [t for c in choices for t in c.get("logprobs", {}).get("tokens", [])]
            assert text == "ab" + REPLY and tokens[:4] == ["a", "b", "H", "i"] and len(tokens) == 2 + len(REPLY.encode())


def test_adapter_by_model_name(server):
    srv, eng = server
    for model, want in (("poetry", "poetry"), ("base", None), ("unknown", None), (None, None)):
        st, data = post(srv, "/v1/completions", {"prompt": "a", "max_tokens": 1, "model": model})
        assert st == 200 and eng.calls[-1]["adapter"] == want
        assert strict(data)["model"] == (want or "base")
    c = http.client.HTTPConnection("127.0.0.1", srv.server_address[1], timeout=10)
    c.request("GET", "/v1/models")
    assert [m["id"] for m in json.loads(c.getresponse().read())["data"]] == ["base", "legal", "poetry"]
    c.close()


@pytest.mark.parametrize("path,extra", [
    ("/v1/completions", {"logprobs": 21}), ("/v1/completions", {"logprobs": -1}), ("/v1/completions", {"logprobs": True}),
    ("/v1/completions", {"logprobs": "3"}), ("/v1/chat/completions", {"logprobs": 3}),
    ("/v1/chat/completions", {"top_logprobs": 2}), ("/v1/chat/completions", {"logprobs": True, "top_logprobs": 21})])
def test_bad_logprobs_are_refused(server, path, extra):
    srv, _ = server
    st, data = post(srv, path, {"prompt": "a", "messages": [{"role": "user", "content": "a"}], "max_tokens": 1, **extra})
    assert st == 400 and "logprobs" in strict(data)["error"]["message"]
