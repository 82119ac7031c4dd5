"""Prompt scoring (moe_head_logprobs) where the candidate lists are put to the test: vocabularies in blocks or
in the order of their logits (a part's list holds 160 entries of its share of the vocabulary), a largest
logit that comes last, and candidates of equal rank in few threads.

Logits here are sums of two bf16 products (a value's leading 8 bits and the next 8): below 2^24 steps of
the smallest bit, so the tensor cores' fp32 sums are exact, and what is left is the arithmetic that the
tolerance of test_gpu_logprobs counts."""
import numpy as np
import pytest
import torch

from test_gpu_logprobs import ATOL, HEAD_TOL, plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch.device("cuda:0")


def two_parts(values):
    hi = values.bfloat16().float()
    return hi, (values - hi).bfloat16().float()


def of_kinds(columns, T, dev):
    """A head [V, 64] with the logits of each kind of row in two columns, rows that pick one kind each in turn,
    and the logits themselves, fp32 [kinds, V]."""
    V = columns[0].numel()
    w, logits = torch.zeros((V, 64)), []
    for k, c in enumerate(columns):
        hi, lo = two_parts(c.float())
        w[:, 2 * k], w[:, 2 * k + 1] = hi, lo
        logits.append((hi.double() + lo.double()).float())
    x = torch.zeros((T, 64))
    kind = torch.arange(T) % len(columns)
    x[torch.arange(T), 2 * kind] = 1.0
    x[torch.arange(T), 2 * kind + 1] = 1.0
    return w.bfloat16().to(dev), x.bfloat16().to(dev), kind, torch.stack(logits).numpy()


def check_kinds(columns, targets, T, n, dev):
    from moe_offload_b200.tokens import head_logprobs
    w, x, kind, logits = of_kinds(columns, T, dev)
    r = head_logprobs(w, x, torch.tensor(targets, dtype=torch.int32)[kind].to(dev), n)
    lp, en, ids, tl = plain(logits, targets, n)
    got = [v.cpu().numpy() for v in (r.logprob, r.entropy, r.top_ids, r.top_logprobs)]
    for t in range(T):
        k = int(kind[t])
        if t >= len(columns):                                # the same row again: the same bits
            for g in got:
                assert np.array_equal(g[t], g[k], equal_nan=True), (t, k)
            continue
        assert np.array_equal(got[2][t], ids[k]), k
        for g, want in ((got[0][t], lp[k]), (got[1][t], en[k]), (got[3][t], tl[k])):
            off = np.abs(g.astype(np.float64) - want)
            assert np.all(off <= ATOL + HEAD_TOL * np.abs(want)), (k, np.max(off / (ATOL + np.abs(want))))


def vocabularies(V):
    """Logits over a vocabulary: rising with a confident last id, in two blocks with one id far above, the same
    without it, rising alone, falling, and a block that all parts meet at their ends."""
    g = torch.Generator().manual_seed(V)
    v = torch.arange(V).float()
    rising = 40.0 * v / V
    last = rising.clone()
    last[V - 1] = 60.0
    blocks = 2.0 * torch.randn(V, generator=g)
    blocks[V * 6 // 10:] += 3.0
    spike = blocks.clone()
    spike[V - V // 30] = 30.0
    ends = 2.0 * torch.randn(V, generator=g)
    ends[V - V // 8:] += 12.0
    return [last, spike, blocks, rising, 40.0 - rising, ends], [V - 1, V - V // 30, V - 5, V - 1, 0, V - 3]


@pytest.mark.parametrize("n", [0, 1, 20, 32])
@pytest.mark.parametrize("T,V", [(1, 80000), (6, 248320), (20, 80000), (128, 50021), (140, 80000), (300, 248320),
                                 (2048, 30000)])
def test_vocabularies_in_order(dev, T, V, n):
    columns, targets = vocabularies(V)
    check_kinds(columns, targets, T, n, dev)


@pytest.mark.parametrize("n", [0, 20])
def test_a_long_prompt_of_a_blocked_vocabulary(dev, n):
    """2,048 rows, 9 parts: a list sees 13,800 entries."""
    columns, targets = vocabularies(248320)
    check_kinds(columns[1:3], targets[1:3], 2048, n, dev)


def test_equal_logits_that_fill_the_lists(dev):
    """Blocks of one value, more than a list holds, with the largest logits behind them."""
    V = 60000
    flat = torch.zeros(V)
    flat[1000:40000] = 2.0
    stairs = torch.div(torch.arange(V), 700, rounding_mode="floor").float()
    one = flat.clone()
    one[V - 1] = 9.0
    for T in (3, 150):
        check_kinds([flat, stairs, one], [0, V - 1, V - 1], T, 20, dev)


def test_one_long_list(dev):
    """A vocabulary of one part: the list alone decides."""
    V = 190
    up = torch.arange(V).float() / 8
    for T in (2, 129):
        check_kinds([up, up.flip(0)], [V - 1, 0], T, 32, dev)


@pytest.mark.parametrize("n", [0, 3, 32])
def test_candidates_crowded_in_few_threads(dev, n):
    """More large logits than are ranked at once, held by fewer threads than alternatives are kept, so that the
    threads' best ones are no bound on them: in each of 27 of a row's 48 lists (one tile of 256 columns a part at
    600 rows of 6,144 logits) the columns that lie 0 to 9 above a multiple of 32 are far above the rest. The 40
    largest come in one of the last lists."""
    V, T = 24 * 256, 600
    v = torch.arange(V)
    lists, lane = torch.div(v, 128, rounding_mode="floor"), v % 32
    high = lists % 16 <= 8
    peak = high & (lane < 10) & ~((lists % 4 == 1) & (lane == 9))
    rng = torch.Generator().manual_seed(40)
    row = torch.where(high, 1.0, 0.0)
    row[peak] = 50.0 + torch.randperm(int(peak.sum()), generator=rng).float() / 256
    best = peak & (lists == 40)
    row[best] = 60.0 + torch.randperm(int(best.sum()), generator=rng).float() / 16
    check_kinds([row], [int(row.argmax())], T, n, dev)
    check_kinds([row], [7], T, n, dev)
