"""Token loop around the MoE stack: embedding lookup, LM head, next-token choice and the
decode loop that drives them (the step after the routed block in the reference:
mlx-qwen38/server.py:93-110 `_sample_next_token`, server.py:113-199 `_generate_stream_impl`,
loader.py:1125-1244 `generate_greedy`).

The reference runs a Qwen3.8 checkpoint's embedding, attention layers and LM head in MLX; none
of them exist here, so `TokenHead.synthetic` builds seeded bf16 tables of the model's shape
(vocabulary V, hidden H) and the loop runs token ids -> embedding rows -> the routed-expert
stack -> LM head -> next id, every step on the GPU through libmoe_b200 (moe_embed_tokens,
moe_lm_head_argmax for greedy steps, moe_lm_head_logits + moe_sample_tokens for sampled ones). `ByteTokenizer` stands in for the tokenizer: ids
0..255 are UTF-8 bytes, `eos_id` ends a generation.
"""
from __future__ import annotations

import time
from typing import Any, Iterable, Iterator, NamedTuple

import torch

from ._lib import call
from .ops import _launch_on, _need, _ptr, _stream

MAX_ALTERNATIVES = 32


class TokenLogprobs(NamedTuple):
    """Per row: the given token's log-probability (NaN where none was given), the entropy in nats,
    and the ids and log-probabilities of the n most likely tokens (most likely first, equal ones
    the lower id first). fp32 [T], fp32 [T], int32 [T, n], fp32 [T, n]."""

    logprob: torch.Tensor | None
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def _logprob_outputs(like: torch.Tensor, T: int, V: int, targets: torch.Tensor | None, n: int) -> TokenLogprobs:
    if not 0 <= n <= min(V, MAX_ALTERNATIVES):
        raise ValueError(f"{n} alternatives: 0 to {min(V, MAX_ALTERNATIVES)} can be asked for")
    if targets is not None:
        _need(targets, "targets", (torch.int32,), like.device)
        if targets.numel() != T:
            raise ValueError(f"{targets.numel()} targets for {T} rows")
    # (new_empty: a third less host time than torch.empty, which parses a device)
    f = torch.float32
    if like.dtype != f:
        return TokenLogprobs(None if targets is None else like.new_empty(T, dtype=f), like.new_empty(T, dtype=f),
                             like.new_empty((T, n), dtype=torch.int32), like.new_empty((T, n), dtype=f))
    return TokenLogprobs(None if targets is None else like.new_empty(T), like.new_empty(T),
                         like.new_empty((T, n), dtype=torch.int32) if targets is None else targets.new_empty((T, n)),
                         like.new_empty((T, n)))


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, n: int = 0,
                   stream=None) -> TokenLogprobs:
    """logits fp32 [T, V], targets int32 [T] (-1: no token) -> TokenLogprobs. A logit of -inf is a
    masked token; a row with a NaN, a +inf or nothing above -inf gives NaN."""
    _need(logits, "logits", (torch.float32,))
    if logits.dim() != 2:
        raise ValueError(f"logits have shape {tuple(logits.shape)}, expected [T, V]")
    T, V = logits.shape
    dev = logits.device
    with _launch_on(dev, stream):
        r = _logprob_outputs(logits, T, V, targets, n)
        if T:
            call("moe_token_logprobs", logits.data_ptr(), T, V, _ptr(targets), n, _ptr(r.logprob),
                 r.entropy.data_ptr(), r.top_ids.data_ptr(), r.top_logprobs.data_ptr(), _stream(stream, dev))
    return r


def head_logprobs(head: torch.Tensor, h: torch.Tensor, targets: torch.Tensor | None = None, n: int = 0,
                  stream=None) -> TokenLogprobs:
    """token_logprobs of the logits of rows h bf16 [T, H] under the head bf16 [V, H], without the
    [T, V] logits in memory (prompt scoring): any T. The alternatives are exact unless a token's sum_h
    |x_h w_vh| is more than four times the largest one's among the row's n + 8 best."""
    _need(head, "head", (torch.bfloat16,))
    dev = head.device
    _need(h, "h", (torch.bfloat16,), dev)
    if head.dim() != 2 or h.dim() != 2 or h.shape[1] != head.shape[1]:
        raise ValueError(f"rows {tuple(h.shape)} do not fit a head {tuple(head.shape)}")
    V, H = head.shape
    T = h.shape[0]
    with _launch_on(dev, stream):
        r = _logprob_outputs(h, T, V, targets, n)
        if T:
            ws = torch.empty(int(call("moe_head_logprobs_workspace_bytes", T, V, n)), dtype=torch.uint8, device=dev)
            call("moe_head_logprobs", head.data_ptr(), V, H, h.data_ptr(), T, _ptr(targets), n, _ptr(r.logprob),
                 r.entropy.data_ptr(), r.top_ids.data_ptr(), r.top_logprobs.data_ptr(), ws.data_ptr(), ws.numel(),
                 _stream(stream, dev))
    return r


class ByteTokenizer:
    """ids 0..255 <-> bytes; eos_id (default V - 1) is the stop token."""

    def __init__(self, vocab_size: int, eos_id: int | None = None):
        if vocab_size < 257:
            raise ValueError("the byte tokenizer needs a vocabulary of at least 257 ids")
        self.vocab_size = vocab_size
        self.eos_token_id = vocab_size - 1 if eos_id is None else int(eos_id)

    def encode(self, text: str) -> list[int]:
        return list(text.encode("utf-8"))

    def decode(self, ids: Iterable[int]) -> str:
        return self.decode_bytes(ids).decode("utf-8", errors="replace")

    def decode_bytes(self, ids: Iterable[int]) -> bytes:
        """What the ids stand for before it is read as text (a token may be part of a character)."""
        return bytes(i for i in ids if 0 <= i < 256)


class TokenHead:
    """Embedding table and LM head, bf16 [V, H] on the device (head None: tied to the embedding)."""

    def __init__(self, embed: torch.Tensor, head: torch.Tensor | None = None):
        _need(embed, "embed", (torch.bfloat16,))
        self.embed_w = embed
        self.head_w = embed if head is None else head
        _need(self.head_w, "head", (torch.bfloat16,), embed.device)
        self.V, self.H = embed.shape
        if tuple(self.head_w.shape) != (self.V, self.H):
            raise ValueError("embedding and head shapes differ")
        self.device = embed.device
        self._ws = None
        self._best = None

    @classmethod
    def synthetic(cls, vocab_size: int, hidden: int, device, seed: int = 7, embed_std: float = 1.0,
                  head_std: float = 0.02) -> "TokenHead":
        """Seeded N(0, embed_std) embedding rows and N(0, head_std) head rows, bf16."""
        dev = torch.device(device)
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        emb = (torch.randn((vocab_size, hidden), generator=g, device=dev) * embed_std).to(torch.bfloat16)
        head = (torch.randn((vocab_size, hidden), generator=g, device=dev) * head_std).to(torch.bfloat16)
        return cls(emb, head)

    @property
    def head_bytes(self) -> int:
        return self.V * self.H * 2

    def embed(self, ids: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """ids int32 [T] (device) -> bf16 [T, H]."""
        _need(ids, "ids", (torch.int32,), self.device)
        T = ids.numel()
        if out is None:
            out = torch.empty((T, self.H), dtype=torch.bfloat16, device=self.device)
        call("moe_embed_tokens", self.embed_w.data_ptr(), self.V, self.H, ids.data_ptr(), T, out.data_ptr(),
             _stream(stream))
        return out

    def logits(self, h: torch.Tensor, out: torch.Tensor | None = None, stream=None, adapters=None,
               adapter_ids: torch.Tensor | None = None) -> torch.Tensor:
        """h bf16 [T, H] (T <= 4) -> fp32 [T, V]. adapters (adapters.AdapterBank of K = H, N = V) with
        adapter_ids int32 [T] (device): each row's low-rank adapter is added, -1 for none."""
        _need(h, "h", (torch.bfloat16,), self.device)
        if adapters is not None and adapter_ids is None:
            raise ValueError("adapters need adapter_ids, one of each row")
        T = h.shape[0]
        if out is None:
            out = torch.empty((T, self.V), dtype=torch.float32, device=self.device)
        call("moe_lm_head_logits", self.head_w.data_ptr(), self.V, self.H, h.data_ptr(), T, out.data_ptr(),
             _stream(stream))
        if adapters is not None:
            adapters.add(out, h, adapter_ids, out=out, stream=stream)
        return out

    def argmax(self, h: torch.Tensor, out: torch.Tensor | None = None, logits: torch.Tensor | None = None,
               stream=None) -> torch.Tensor:
        """h bf16 [T, H] -> int32 [T] greedy next ids, the LM head and the argmax in one pass
        (logits, when given, also receives the fp32 logits)."""
        _need(h, "h", (torch.bfloat16,), self.device)
        T = h.shape[0]
        if out is None:
            out = torch.empty((T,), dtype=torch.int32, device=self.device)
        need = int(call("moe_lm_head_argmax_workspace_bytes", T))
        if self._best is None or self._best.numel() * 8 < need:
            self._best = torch.zeros(max(4, T), dtype=torch.int64, device=self.device)
        call("moe_lm_head_argmax", self.head_w.data_ptr(), self.V, self.H, h.data_ptr(), T,
             None if logits is None else logits.data_ptr(), out.data_ptr(), self._best.data_ptr(),
             self._best.numel() * 8, _stream(stream))
        return out

    def score(self, h: torch.Tensor, targets: torch.Tensor | None = None, n: int = 0, stream=None) -> TokenLogprobs:
        """h bf16 [T, H], targets int32 [T] -> TokenLogprobs under this head (head_logprobs)."""
        _need(h, "h", (torch.bfloat16,), self.device)
        return head_logprobs(self.head_w, h, targets, n, stream=stream)

    def sample(self, logits: torch.Tensor, temperature: float = 0.0, top_p: float = 1.0, seed: int = 0,
               counter: int = 0, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """fp32 [T, V] -> int32 [T] next ids (argmax when temperature <= 0)."""
        _need(logits, "logits", (torch.float32,), self.device)
        T, V = logits.shape
        if out is None:
            out = torch.empty((T,), dtype=torch.int32, device=self.device)
        need = int(call("moe_sample_workspace_bytes", T, V))
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        call("moe_sample_tokens", logits.data_ptr(), T, V, float(temperature), float(top_p),
             int(seed) & 0xFFFFFFFFFFFFFFFF, int(counter) & 0xFFFFFFFFFFFFFFFF, out.data_ptr(), self._ws.data_ptr(),
             self._ws.numel(), _stream(stream))
        return out


def _records(ids: list[int], r: TokenLogprobs) -> list[dict[str, Any]]:
    """One host record per row: id, logprob, entropy, top [(id, logprob), ..] (a read of the device)."""
    lp, ent = r.logprob.tolist(), r.entropy.tolist()
    ti, tl = r.top_ids.tolist(), r.top_logprobs.tolist()
    return [{"id": i, "logprob": lp[t], "entropy": ent[t], "top": list(zip(ti[t], tl[t]))} for t, i in enumerate(ids)]


def score_prompt(head: TokenHead, rows: torch.Tensor, prompt_ids: list[int], n: int = 0, adapters=None,
                 adapter: int = -1) -> list[dict[str, Any]]:
    """Records of prompt_ids[1:], each under the row before it: rows bf16 [len(prompt_ids), H] are the stack's
    outputs. With an adapter the logits come four rows at a time (TokenHead.logits); without one straight
    from the rows (TokenHead.score)."""
    if len(prompt_ids) < 2:
        return []
    ids = torch.tensor(list(prompt_ids[1:]), dtype=torch.int32).to(head.device, non_blocking=True)
    if adapters is None or adapter < 0:
        return _records(list(prompt_ids[1:]), head.score(rows[:-1].contiguous(), ids, n))
    of = torch.full((4,), adapter, dtype=torch.int32, device=head.device)
    out: list[dict[str, Any]] = []
    for t in range(0, len(prompt_ids) - 1, 4):
        m = min(4, len(prompt_ids) - 1 - t)
        logits = head.logits(rows[t:t + m].contiguous(), adapters=adapters, adapter_ids=of[:m])
        out += _records(list(prompt_ids[1 + t:1 + t + m]), token_logprobs(logits, ids[t:t + m], n))
    return out


def generate_stream(stack, head: TokenHead, prompt_ids: list[int], max_tokens: int, temperature: float = 0.0,
                    top_p: float = 1.0, stop_ids: Iterable[int] | None = None, seed: int = 0,
                    timings: dict[str, Any] | None = None, adapters=None, adapter: int = -1,
                    logprobs: int | None = None, scored: list | None = None,
                    prompt_scored: list | None = None) -> Iterator[int]:
    """server.py:113-199 as a token-id generator over `stack` (anything with prefill(rows [T, H])
    -> [T, H] and decode_token(h [1, H]) -> [1, H], e.g. offload.OffloadStack): prefill of the
    prompt's embedding rows, the next id from the last row's logits, then one decode step per
    yielded id until max_tokens, a stop id, or the caller stops iterating. `timings` receives
    prefill_s, decode_s, decode_tok_per_s, stopped_by_token (the reference's keys). Each step
    reads its id back to the host (the stop test), as the reference does.

    adapters / adapter: a bank of low-rank adapters on the LM head and the one this generation uses
    (-1: none). logprobs = n: `scored` receives a record of every yielded id before it is yielded (id,
    logprob, entropy, top: the n most likely ids with their log-probabilities, of the distribution
    before temperature and top_p), and `prompt_scored`, when given, those of prompt_ids[1:]."""
    stop_set = set(int(x) for x in stop_ids) if stop_ids is not None else set()
    tm = timings if timings is not None else {}
    tm.update({"prefill_s": 0.0, "decode_s": 0.0, "decode_tok_per_s": 0.0, "stopped_by_token": False})
    if max_tokens <= 0:
        return
    if not prompt_ids:
        raise ValueError("empty prompt")
    if adapters is not None and not -1 <= adapter < adapters.adapters:
        raise ValueError(f"adapter {adapter}: the bank has {adapters.adapters}")
    if adapters is None and adapter >= 0:
        raise ValueError(f"adapter {adapter}: there is no bank of adapters")
    dev = head.device
    t0 = time.perf_counter()
    bank = adapters if adapter >= 0 else None
    of = None if bank is None else torch.full((1,), adapter, dtype=torch.int32).to(dev)
    ids = torch.tensor(list(prompt_ids), dtype=torch.int32).to(dev, non_blocking=True)
    rows = head.embed(ids)
    out = stack.prefill(rows)
    greedy = not temperature > 0.0
    # the fused head and argmax leave no logits to adapt or score
    fused = greedy and bank is None and logprobs is None
    logits = head.logits(out[-1:].contiguous(), adapters=bank, adapter_ids=of)
    cur = head.sample(logits, temperature, top_p, seed, 0)
    tok = int(cur.item())
    if logprobs is not None and prompt_scored is not None:
        prompt_scored += score_prompt(head, out, list(prompt_ids), logprobs, bank, adapter)
    tm["prefill_s"] = round(time.perf_counter() - t0, 4)
    n = 0
    t_dec0 = time.perf_counter()
    try:
        for d in range(max_tokens):
            if tok in stop_set:
                tm["stopped_by_token"] = True
                break
            n += 1
            if logprobs is not None and scored is not None:
                scored += _records([tok], token_logprobs(logits, cur, logprobs))
            yield tok
            if d + 1 >= max_tokens:
                break
            y = stack.decode_token(head.embed(cur))
            if fused:
                head.argmax(y, out=cur)
            else:
                head.logits(y, out=logits, adapters=bank, adapter_ids=of)
                head.sample(logits, temperature, top_p, seed, d + 1, out=cur)
            tok = int(cur.item())
    finally:
        dec = max(1e-6, time.perf_counter() - t_dec0)
        tm["decode_s"] = round(dec, 4)
        tm["decode_tok_per_s"] = round(n / dec, 3)


class ResidentTokenLoop:
    """Greedy / sampled decode over a resident stack.PersistentStack, one CUDA graph per token:
    embedding row -> the persistent stack launch -> LM head -> next id, with the id copied to a
    pinned host word (the only per-token transfer). `step()` returns that id."""

    def __init__(self, stack, head: TokenHead, temperature: float = 0.0, top_p: float = 1.0, seed: int = 0):
        self.stack, self.head = stack, head
        self.temperature, self.top_p, self.seed = float(temperature), float(top_p), int(seed)
        dev = head.device
        self.cur = torch.zeros((1,), dtype=torch.int32, device=dev)
        self.logits = torch.empty((1, head.V), dtype=torch.float32, device=dev)
        self.host_id = torch.zeros((1,), dtype=torch.int32, pin_memory=True)
        self.counter = 0
        self.graph = None
        self._graph_failed = False
        # embed, stack, head (+ the argmax's id kernel when greedy) / head + sample
        self.launches_per_step = 4

    def _body(self) -> None:
        self.head.embed(self.cur, out=self.stack.x_in)
        self.stack.step_device()
        if self.temperature <= 0.0:
            self.head.argmax(self.stack.y, out=self.cur)
        else:
            # the counter of a captured step would be fixed at capture: a sampled loop runs uncaptured
            self.head.logits(self.stack.y, out=self.logits)
            self.head.sample(self.logits, self.temperature, self.top_p, self.seed, self.counter, out=self.cur)
        self.host_id.copy_(self.cur, non_blocking=True)

    def start(self, token_id: int) -> None:
        self.cur.fill_(int(token_id))
        self.counter = 0

    def _capture(self) -> None:
        cur = torch.cuda.current_stream(self.head.device)
        s = torch.cuda.Stream(device=self.head.device)
        s.wait_stream(cur)
        try:
            with torch.cuda.stream(s):
                save = self.cur.clone()
                self._body()                                      # warm-up outside the graph
                self.cur.copy_(save)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                self._body()
            self.graph = g
        except RuntimeError:
            # a driver that cannot capture the cooperative stack launch: run the step directly
            self._graph_failed = True
            torch.cuda.synchronize(self.head.device)
        cur.wait_stream(s)

    def step(self) -> int:
        self.counter += 1
        if self.temperature <= 0.0 and self.graph is None and not self._graph_failed:
            self._capture()
        if self.temperature <= 0.0 and self.graph is not None:
            self.graph.replay()
        else:
            self._body()
        torch.cuda.current_stream(self.head.device).synchronize()
        return int(self.host_id.item())
