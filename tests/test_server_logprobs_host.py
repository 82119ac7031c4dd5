"""The server's `logprobs` where tokens are no text of their own: parts of a character, ids without bytes, ids of
equal text. Over the stand-in engine, without a GPU."""
import threading

import pytest

from test_answering_host import Engine, post, strict


@pytest.fixture()
def serve():
    from moe_offload_b200.server import make_server
    running = []

    def start(engine):
        srv = make_server(engine, "127.0.0.1", 0, model_id="base", default_max_tokens=64)
        threading.Thread(target=srv.serve_forever, daemon=True).start()
        running.append(srv)
        return srv
    yield start
    for srv in running:
        srv.shutdown()
        srv.server_close()


class Says(Engine):
    """Answers with the given ids, whatever is asked."""

    def __init__(self, ids):
        super().__init__()
        self.ids = ids

    def generate_stream(self, prompt_ids, max_tokens, temperature=0.0, top_p=1.0, stop_ids=None, seed=0, adapter=None,
                        logprobs=None, scored=None, prompt_scored=None):
        if prompt_scored is not None:
            prompt_scored += [self.record(i, logprobs) for i in prompt_ids[1:]]
        for i in self.ids[:max_tokens]:
            if logprobs is not None:
                scored.append(self.record(i, logprobs))
            yield i


def chat(srv, **more):
    body = {"messages": [{"role": "user", "content": "x"}], "max_tokens": 40, "logprobs": True, **more}
    st, data = post(srv, "/v1/chat/completions", body)
    assert st == 200
    return strict(data)["choices"][0]["logprobs"]["content"]


def test_bytes_of_parts_of_a_character(serve):
    """Put together, the tokens' bytes are the answer's, whatever the tokens' texts."""
    text = "\xe9 €\U0001f600."
    content = chat(serve(Says(list(text.encode()))))
    assert b"".join(bytes(c["bytes"]) for c in content).decode() == text
    assert content[0]["bytes"] == [195] and content[0]["token"] == "token_id:195"


def test_bytes_of_an_id_without_any(serve):
    """An id that stands for no bytes has none: null, as the interface has it."""
    content = chat(serve(Says([65, 298])), top_logprobs=2)
    assert content[1]["token"] == "token_id:298" and content[1]["bytes"] is None
    assert content[1]["top_logprobs"][0]["bytes"] is None and content[0]["bytes"] == [65]
