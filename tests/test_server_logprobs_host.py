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


def completion(srv, **more):
    st, data = post(srv, "/v1/completions", {"max_tokens": 40, "logprobs": 0, **more})
    assert st == 200
    return strict(data)["choices"][0]


TEXT = "a\xe9b€\U0001f600.c"


def places(text):
    """Where in the text each byte's character stands."""
    return [k for k, c in enumerate(text) for _ in c.encode()]


def test_offsets_of_parts_of_a_character(serve):
    choice = completion(serve(Says(list(TEXT.encode()))), prompt="x")
    assert choice["text"] == TEXT and choice["logprobs"]["text_offset"] == places(TEXT)


def test_offsets_behind_an_echoed_prompt(serve):
    choice = completion(serve(Says(list(TEXT.encode()))), prompt="€ x\xe9", echo=True)
    assert choice["text"] == "€ x\xe9" + TEXT and choice["logprobs"]["text_offset"] == places("€ x\xe9" + TEXT)


@pytest.mark.parametrize("echo", [False, True])
def test_offsets_of_a_stream(serve, echo):
    srv = serve(Says(list(TEXT.encode())))
    st, data = post(srv, "/v1/completions", {"prompt": "\xe9€", "max_tokens": 40, "logprobs": 0, "echo": echo, "stream": True})
    choices = [strict(e[6:])["choices"][0] for e in data.decode().split("\n\n") if e.startswith("data: {")]
    text = "".join(c["text"] for c in choices)
    offsets = [o for c in choices for o in c.get("logprobs", {}).get("text_offset", [])]
    assert text == ("\xe9€" if echo else "") + TEXT and offsets == places(text)


def test_offsets_of_bytes_that_are_no_text(serve):
    """Bytes that begin no character, or one that does not come: a replacement character each, and what follows
    them stands behind those."""
    ids = [0xe9, 0x28, 0xff, 0x80, 0x41, 298, 0x42, 0xe2, 0x82]
    choice = completion(serve(Says(ids)), prompt="x")
    assert choice["text"] == "�(��AB�"
    got = choice["logprobs"]["text_offset"]
    assert [got[ids.index(i)] for i in (0x28, 0x41, 0x42, 0xe2, 0x82)] == [1, 4, 5, 6, 6]
    assert got == sorted(got)


class OneText(Says):
    """A vocabulary in which 66 and 67 read alike (as words with and without a leading space do in many)."""

    def __init__(self, ids):
        super().__init__(ids)
        inner = self.tokenizer

        class Tokenizer:
            eos_token_id = inner.eos_token_id

            def encode(self, text):
                return inner.encode(text)

            def decode(self, ids):
                return inner.decode([66 if i == 67 else i for i in ids])

        self.tokenizer = Tokenizer()


def test_alternatives_of_equal_text(serve):
    """Each alternative has its place: a second one of the same text goes by its number."""
    choice = completion(serve(OneText([65])), prompt="x", logprobs=3)
    assert choice["logprobs"]["top_logprobs"] == [{"A": 0.0, "B": -0.25, "token_id:67": None}]
    choice = completion(serve(OneText([66])), prompt="x", logprobs=2)
    assert choice["logprobs"]["top_logprobs"] == [{"B": 0.0, "token_id:67": -0.25}]
