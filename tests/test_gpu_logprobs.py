"""Log-probabilities of given tokens, entropy and alternatives (moe_token_logprobs,
moe_head_logprobs) against the definition in 64 bits.

Tolerances. With m the row's largest logit and s = sum of the other e^(x - m), lse - m = log1p(s).
An exponent's argument x - m is rounded once (2^-24 relative) and multiplied by log2(e) (2^-24
relative again), so e^(x - m) is off by at most |x - m| * 2^-23 relative, plus 2^-22 of the hardware
exponential; terms with |x - m| > 30 carry less than 1e-13 of the weight. A thread adds at most
V / 512 <= 485 terms, one after another, and 14 merges follow: 499 * 2^-24 = 3e-5 if all roundings had
one sign. So s is off by at most 30 * 2^-23 + 2^-22 + 3e-5 < 4e-5 relative, and log1p(s) by no more,
since s / (1 + s) <= log1p(s). A log-probability is (x - m) - log1p(s) with both terms <= 0, the entropy
log1p(s) - w / (1 + s) with both terms >= 0: neither cancels, so the relative bound carries over to
them. RTOL = 5e-5; ATOL covers results below the smallest normal fp32 number."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ATOL, RTOL = 1e-37, 5e-5


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch.device("cuda:0")


def ordered(l, n):
    """ids of the n largest values of a row, equal ones the lower id first, NaN as -inf."""
    l = np.where(np.isnan(l), -np.inf, l) + 0.0
    return np.lexsort((np.arange(l.size), -l))[:n]


def plain(logits, targets, n):
    """(logprob, entropy, top ids, top logprobs) of fp32 logits [T, V], in 64 bits."""
    T = logits.shape[0]
    lp, en = np.full(T, np.nan), np.full(T, np.nan)
    ids, tl = np.zeros((T, n), np.int64), np.full((T, n), np.nan)
    for t in range(T):
        l = logits[t].astype(np.float64)
        ids[t] = ordered(logits[t], n)
        m = np.max(l)                                     # NaN if there is one
        if not np.isfinite(m):
            continue
        with np.errstate(divide="ignore", invalid="ignore"):
            z = l - m
            e = np.exp(z)
            first = int(np.argmax(l))
            e[first] = 0.0
            rest = e.sum()
            lse = np.log1p(rest)
            en[t] = lse - np.where(e > 0, e * z, 0.0).sum() / (1.0 + rest)
        if targets is not None and targets[t] >= 0:
            lp[t] = z[targets[t]] - lse
        tl[t] = z[ids[t]] - lse
    return lp, en, ids, tl


def close(got, want, what):
    got = got.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got == -np.inf, want == -np.inf), what
    ok = np.isfinite(want)
    off = np.abs(got[ok] - want[ok])
    assert np.all(off <= ATOL + RTOL * np.abs(want[ok])), (what, np.max(off / (ATOL + np.abs(want[ok]))))


def check(logits, targets, n, dev):
    from moe_offload_b200.tokens import token_logprobs
    r = token_logprobs(torch.from_numpy(logits).to(dev),
                       None if targets is None else torch.from_numpy(np.asarray(targets, np.int32)).to(dev), n)
    lp, en, ids, tl = plain(logits, targets, n)
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    close(r.entropy, en, "entropy")
    close(r.top_logprobs, tl, "top_logprobs")
    if targets is None:
        assert r.logprob is None
    else:
        close(r.logprob, lp, "logprob")
    return r


@pytest.mark.parametrize("T,V,n", [(1, 1, 0), (1, 1, 1), (2, 2, 2), (3, 3, 1), (5, 31, 31), (4, 32, 32), (4, 33, 32),
                                   (7, 257, 5), (2, 511, 20), (2, 2047, 32), (3, 4099, 20), (1, 8193, 7),
                                   (1, 32771, 32), (1, 248320, 20), (3, 50021, 1), (300, 1000, 3), (600, 9001, 2)])
def test_against_definition(dev, T, V, n):
    rng = np.random.default_rng(T * 1000 + V + n)
    lg = rng.normal(0, 3, (T, V)).astype(np.float32)
    targets = rng.integers(0, V, T)
    targets[T // 2] = -1
    check(lg, targets, n, dev)
    check(lg, None, n, dev)


@pytest.mark.parametrize("V", [5, 257, 4099, 70001])
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "two values"])
def test_orders_and_ties(dev, V, order):
    """Sorted rows (every element a new maximum, or none) and ties, which go to the lower id."""
    n = min(V, 32)
    i = np.arange(V, dtype=np.float32)
    row = {"rising": i / 7, "falling": -i / 7, "equal": np.full(V, -3.25, np.float32),
           "two values": np.where(np.random.default_rng(V).random(V) < 0.2, 1.5, -0.0).astype(np.float32)}[order]
    check(np.stack([row, row[::-1], np.roll(row, 1)]).astype(np.float32), [0, V - 1, V // 2], n, dev)


@pytest.mark.parametrize("V", [4096, 50021, 248320])
def test_large_values_crowded(dev, V):
    """Large elements that crowd into one residue, one thread's share or one end of the row."""
    rng = np.random.default_rng(V)
    lg = rng.normal(0, 1, (6, V)).astype(np.float32)
    lg[0, ::32] += 50                                     # one residue mod 32, more than are ranked at once
    lg[1, 5::2048] += 50
    lg[2, :700] += 50
    lg[3, -700:] += 50
    lg[4, ::32] = 9.0                                     # ties there
    lg[5, 3::64] = np.arange(lg[5, 3::64].size, dtype=np.float32)
    for n in (1, 5, 20, 32):
        check(lg, [0, 5, 6, V - 1, 32, 3], n, dev)


def test_zero_signs_tie(dev):
    lg = np.array([[-0.0, 0.0, -0.0, 0.0, -1.0]], np.float32)
    check(lg, [1], 5, dev)


@pytest.mark.parametrize("V,left", [(300, 1), (300, 3), (50021, 1), (50021, 12), (248320, 40)])
def test_masked_rows(dev, V, left):
    """A mask that leaves a few tokens: the alternatives go on with masked ids in order, at -inf."""
    rng = np.random.default_rng(V + left)
    lg = np.full((3, V), -np.inf, np.float32)
    keep = [np.sort(rng.choice(V, left, replace=False)) for _ in range(3)]
    for t in range(3):
        lg[t, keep[t]] = rng.normal(0, 2, left)
    masked = int(np.setdiff1d(np.arange(V), keep[1])[0])
    check(lg, [int(keep[0][0]), masked, int(keep[2][-1])], 20, dev)


def test_lowest_value_is_a_number(dev):
    """A mask of the type's lowest value is not -inf: finite log-probabilities far below."""
    low = np.finfo(np.float32).min
    lg = np.full((2, 4100), low, np.float32)
    lg[0, 17] = 1.0
    r = check(lg[1:], [5], 3, dev)                        # all equal: a uniform row
    assert abs(float(r.logprob[0]) + math.log(4100)) < 5e-4
    from moe_offload_b200.tokens import token_logprobs
    r = token_logprobs(torch.from_numpy(lg[:1]).to(dev), torch.tensor([17], dtype=torch.int32, device=dev), 3)
    assert float(r.logprob[0]) == 0.0 and float(r.entropy[0]) == 0.0
    assert r.top_ids[0].tolist() == [17, 0, 1]


@pytest.mark.parametrize("V", [6, 257, 9001])
def test_rows_without_a_distribution(dev, V):
    """All masked, a NaN, a +inf: NaN everywhere, ids still in order; the rows beside them are not touched."""
    rng = np.random.default_rng(V)
    lg = rng.normal(0, 2, (7, V)).astype(np.float32)
    lg[0] = -np.inf
    lg[2, V // 2] = np.nan
    lg[3, 1] = np.inf
    lg[4] = np.nan
    lg[5, :] = -np.inf
    lg[5, V - 1] = np.nan
    check(lg, [0, 1, 2, 1, 3, 4, 5], min(V, 6), dev)


def test_peaked_rows_keep_their_digits(dev):
    """A target whose probability is all but one: its log-probability is -s, far below 2^-24."""
    V = 20011
    rng = np.random.default_rng(3)
    lg = rng.normal(0, 1, (12, V)).astype(np.float32)
    tgt = rng.integers(0, V, 12)
    for t in range(12):
        lg[t, tgt[t]] = 12.0 + 6 * t
    r = check(lg, tgt, 4, dev)
    assert float(r.logprob[11]) < 0.0


def test_bad_target_flagged(dev):
    from moe_offload_b200 import _lib
    from moe_offload_b200.tokens import token_logprobs
    lg = torch.randn((3, 100), device=dev)
    _lib.call("moe_device_error", 1)
    r = token_logprobs(lg, torch.tensor([100, -1, 99], dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    assert int(_lib.call("moe_device_error", 1)) & 2
    assert torch.isnan(r.logprob).tolist() == [True, True, False]
    token_logprobs(lg, torch.tensor([0, -1, 99], dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    assert int(_lib.call("moe_device_error", 1)) == 0


def test_unaligned_rows_and_views(dev):
    """Rows at any 4-byte offset (a view into a larger buffer), nothing written around the outputs."""
    from moe_offload_b200.tokens import token_logprobs
    rng = np.random.default_rng(8)
    for off in range(4):
        for V in (1, 2, 5, 1023, 4097):
            buf = torch.from_numpy(rng.normal(0, 2, 3 * V + 8).astype(np.float32)).to(dev)
            lg = buf[off:off + 3 * V].view(3, V)
            n = min(V, 4)
            r = token_logprobs(lg, torch.zeros(3, dtype=torch.int32, device=dev), n)
            lp, en, ids, tl = plain(lg.cpu().numpy(), [0, 0, 0], n)
            assert np.array_equal(r.top_ids.cpu().numpy(), ids)
            close(r.logprob, lp, "logprob")
            close(r.entropy, en, "entropy")


def test_empty_batch(dev):
    from moe_offload_b200.tokens import head_logprobs, token_logprobs
    none = torch.empty((0,), dtype=torch.int32, device=dev)
    r = token_logprobs(torch.empty((0, 50), device=dev), none, 3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
    r = head_logprobs(torch.empty((50, 64), dtype=torch.bfloat16, device=dev),
                      torch.empty((0, 64), dtype=torch.bfloat16, device=dev), none, 3)
    assert r.entropy.shape == (0,) and r.top_logprobs.shape == (0, 3)


def test_captured_and_on_another_stream(dev):
    """The same bits eagerly, on a side stream and replayed from a graph with new logits."""
    from moe_offload_b200.tokens import token_logprobs
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    lg = torch.randn((3, 70001), generator=g, device=dev) * 3
    tg = torch.randint(0, 70001, (3,), generator=g, device=dev, dtype=torch.int32)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    side = token_logprobs(lg, tg, 20, stream=s)
    s.synchronize()
    want = token_logprobs(lg, tg, 20)
    for a, b in zip(side, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(lg, tg, 20)
    for k in range(3):
        lg.copy_(torch.randn((3, 70001), generator=g, device=dev))
        graph.replay()
        want = token_logprobs(lg, tg, 20)
        for a, b in zip(out, want):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ from hidden rows and the head

def head_case(dev, T, V, H, seed, lean=0.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    w = (torch.randn((V, H), generator=g, device=dev) * 0.02 * (2048 / H) ** 0.5).to(torch.bfloat16)
    tg = torch.randint(0, V, (T,), generator=g, device=dev, dtype=torch.int32)
    x = torch.randn((T, H), generator=g, device=dev)
    x = (x + lean * w[tg.long()].float()).to(torch.bfloat16)
    return w, x, tg


def exact_logits(w, x):
    return torch.matmul(x.double(), w.double().t()).float().cpu().numpy()


# The head form's other logits may be sums of H bf16 products in fp32 on the tensor cores: each of the
# H / 16 steps may drop up to 2^-23 of the running sum, so a logit of size L is off by at most
# L * H / 16 * 2^-23: 1.2e-4 for H = 2048 and L = 8. The log of the sum of e^logit moves by no more
# than their mean error, weighted by probability, and the many steps of smaller partial sums leave
# less than that; targets and alternatives themselves are summed in 64 bits.
HEAD_TOL = 1e-4


def check_head(w, x, tg, n):
    from moe_offload_b200.tokens import head_logprobs
    r = head_logprobs(w, x, tg, n)
    lp, en, ids, tl = plain(exact_logits(w, x), None if tg is None else tg.cpu().numpy(), n)
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    for got, want in ((r.logprob, lp), (r.entropy, en), (r.top_logprobs, tl)):
        if got is None:
            continue
        got = got.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        ok = np.isfinite(want)
        off = np.abs(got[ok] - want[ok])
        assert np.all(off <= ATOL + HEAD_TOL * np.abs(want[ok])), np.max(off / (ATOL + np.abs(want[ok])))
    return r


@pytest.mark.parametrize("T,V,H,n", [(1, 1, 8, 1), (1, 2, 8, 2), (1, 300, 64, 5), (2, 257, 72, 20), (3, 255, 136, 0),
                                     (5, 1000, 1024, 32), (17, 4097, 520, 20), (127, 769, 256, 3), (128, 1024, 256, 20),
                                     (129, 513, 264, 5), (256, 2048, 128, 8), (257, 50021, 64, 20),
                                     (300, 33, 512, 32), (33, 32003, 2048, 0), (1, 248320, 1024, 20),
                                     (640, 5000, 768, 20),
                                     (2049, 700, 64, 5), (2500, 1300, 72, 3), (6, 400, 8192, 4), (130, 512, 64, 32),
                                     (40, 513, 64, 32)])
def test_head_against_definition(dev, T, V, H, n):
    w, x, tg = head_case(dev, T, V, H, T + V + H)
    tg[T // 2] = -1
    check_head(w, x, tg, n)
    check_head(w, x, None, n)


def test_lm_head_rows_at_the_shared_memory_border(dev):
    """T * H = 12,288: the staged rows alone are 48 KB, with the kernel's own arrays more."""
    from moe_offload_b200.tokens import TokenHead
    w, x, _ = head_case(dev, 6, 500, 2048, 21)
    assert np.array_equal(TokenHead(w).logits(x[:4]).cpu().numpy(), exact_logits(w, x[:4]))
    w, x, _ = head_case(dev, 4, 500, 3072, 22)
    assert np.array_equal(TokenHead(w).logits(x).cpu().numpy(), exact_logits(w, x))


def test_head_peaked_rows(dev):
    w, x, tg = head_case(dev, 40, 9000, 1024, 4, lean=30.0)
    r = check_head(w, x, tg, 6)
    assert float(r.logprob.max()) > -1e-3


@pytest.mark.parametrize("T,V,H,n", [(2, 3006, 64, 5), (140, 3006, 64, 5), (600, 20000, 64, 5), (1100, 9000, 64, 3),
                                     (2048, 5000, 64, 0), (2048, 5000, 64, 1)])
def test_head_negative_logits(dev, T, V, H, n):
    """Rows whose logits are all negative, at numbers of lists (two a part) below the 64 sets that bound
    the candidates: a set without a list must count for nothing."""
    w, x, tg = head_case(dev, T, V, H, T + V)
    w[:, 0] = -8.0
    x[:, 0] = 3.0
    for k in range(2):                           # (the second run meets other leftovers in shared memory)
        check_head(w, x, tg, n)


def test_head_cancelling_leaders(dev):
    """The leading logits are sums that cancel to 0 and that the tensor cores leave a little beside it: their
    errors are no share of their size, and the entries at -10 (a fifth of the sum) must not be moved by one.
    The 13 = n + 8 leading ones are summed again exactly and the others are single products, so what is left is
    the arithmetic that HEAD_TOL counts."""
    V, H, n = 60000, 1024, 5
    g = torch.Generator().manual_seed(77)
    w = torch.zeros((V, H))
    w[:, 0] = -10.0
    half = torch.randn((n + 8, H // 2), generator=g) * 2.0 ** torch.randint(-14, 7, (n + 8, H // 2), generator=g)
    half = half.bfloat16().float()
    w[100:100 + n + 8] = torch.cat((half, -half.flip(1)), 1)
    w = w.bfloat16().to(dev)
    for T in (1, 3, 140):
        x = torch.ones((T, H), dtype=torch.bfloat16, device=dev)
        check_head(w, x, torch.arange(T, dtype=torch.int32, device=dev) + 99, n)


@pytest.mark.parametrize("size", [1e3, 2.0 ** 20, -2.0 ** 20, 2.0 ** 29])
def test_head_large_logits(dev, size):
    """Logits of a large size, each a single product (the tensor cores lose nothing): 6 equal ones and
    3,000 that lie a step of bf16 below, or all equal. What lies below is nothing next to them, the equal
    ones' log-probability is -log of their number."""
    V, H = 3006, 64
    for equal in (6, V):
        w = torch.zeros((V, H))
        w[:, 0] = size * (0.5 if size > 0 else 2.0)
        w[1000:1006, 0] = size
        if equal == V:
            w[:, 0] = size
        x = torch.zeros((2, H))
        x[:, 0] = 1.0
        check_head(w.bfloat16().to(dev), x.bfloat16().to(dev), torch.tensor([1002, 1005], dtype=torch.int32, device=dev), 5)


def test_head_ties_and_padding_rows(dev):
    """Equal head rows (more than can be alternatives), rows of zeros (a padded batch: every logit
    equal), and the ids still the lowest first."""
    w, x, tg = head_case(dev, 70, 3001, 256, 9)
    w[100:180] = w[7]
    w[2900:2990] = w[7]
    x[3] = 0
    x[40:60] = 0
    x[5] = (30 * w[7].float()).to(torch.bfloat16)
    x[6] = (-30 * w[7].float()).to(torch.bfloat16)
    check_head(w, x, tg, 20)
    check_head(w, x, tg, 32)


@pytest.mark.parametrize("T", [1, 2, 9, 40, 150])
def test_head_near_ties(dev, T):
    """Logits closer together than fp32 sums tell apart: the order is that of the 64-bit sums."""
    g = torch.Generator(device=dev)
    g.manual_seed(12)
    H, V = 2048, 2000
    base = torch.randn((1, H), generator=g, device=dev)
    w = (base * 0.02).to(torch.bfloat16).repeat(V, 1)
    # each row differs from the others in the last bit of a few of its smallest entries
    small = base[0].abs().argsort()[:64]
    pick = torch.randint(0, 64, (V,), generator=g, device=dev)
    rows = torch.arange(V, device=dev)
    col = small[pick]
    w[rows, col] = (w[rows, col].float() * (1 + 2.0 ** -7)).to(torch.bfloat16)
    x = (base + 0.05 * torch.randn((T, H), generator=g, device=dev)).to(torch.bfloat16)
    check_head(w, x, torch.zeros(T, dtype=torch.int32, device=dev), 20)


def test_head_rows_without_a_distribution(dev):
    w, x, tg = head_case(dev, 10, 700, 128, 13)
    x[2, 5] = float("nan")
    x[7, 0] = float("inf")
    from moe_offload_b200.tokens import head_logprobs
    r = head_logprobs(w, x, tg, 4)
    lg = exact_logits(w, x)
    lp, en, ids, tl = plain(lg, tg.cpu().numpy(), 4)
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    assert np.array_equal(np.isnan(r.logprob.cpu().numpy()), np.isnan(lp))
    assert np.array_equal(np.isnan(r.entropy.cpu().numpy()), np.isnan(en))
    assert np.array_equal(np.isnan(r.top_logprobs.cpu().numpy()), np.isnan(tl))


def test_head_bad_target_flagged(dev):
    from moe_offload_b200 import _lib
    from moe_offload_b200.tokens import head_logprobs
    w, x, _ = head_case(dev, 3, 300, 64, 14)
    _lib.call("moe_device_error", 1)
    r = head_logprobs(w, x, torch.tensor([300, -1, 299], dtype=torch.int32, device=dev), 2)
    torch.cuda.synchronize()
    assert int(_lib.call("moe_device_error", 1)) & 2
    assert torch.isnan(r.logprob).tolist() == [True, True, False]


def test_head_captured_graphs_and_streams(dev):
    """Two captured graphs and an eager call in turn, and two streams at once: the same bits."""
    from moe_offload_b200.tokens import TokenHead
    w, x, tg = head_case(dev, 150, 9001, 256, 15)
    head = TokenHead(w)
    want = head.score(x, tg, 20)
    graphs = []
    for rows in (x, x[:37].contiguous()):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = head.score(rows, tg[:rows.shape[0]].contiguous(), 20)
        graphs.append((gr, out, rows.shape[0]))
    for _ in range(2):
        for gr, out, m in graphs:
            gr.replay()
            for a, b in zip(out, want):
                if m == 150:
                    assert torch.equal(a, b[:m])
                else:
                    assert torch.allclose(a.double(), b[:m].double(), rtol=HEAD_TOL, atol=1e-6)
    s1, s2 = torch.cuda.Stream(device=dev), torch.cuda.Stream(device=dev)
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream(dev))
    outs = [head.score(x, tg, 20, stream=s) for s in (s1, s2) for _ in range(3)]
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, want):
            assert torch.equal(a, b)


def test_head_same_bits_every_time(dev):
    """What the parts of the vocabulary tell each other while they run does not show in the results."""
    from moe_offload_b200.tokens import head_logprobs
    for T, V, H in ((700, 20000, 128), (64, 60000, 64)):
        w, x, tg = head_case(dev, T, V, H, 31)
        w[5000:5200] = w[17]
        x[3] = 0                                             # a padded row: every logit equal
        want = head_logprobs(w, x, tg, 20)
        assert want.top_ids[3].tolist() == list(range(20))
        for _ in range(6):
            for a, b in zip(head_logprobs(w, x, tg, 20), want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("order", [1, -1])
def test_head_rising_and_falling(dev, order):
    """Head rows in the order of their logits: every tile above (or below) all before it, so that no
    bound taken on the way helps."""
    T, V, H = 20, 80000, 64
    g = torch.Generator(device=dev)
    g.manual_seed(32)
    base = torch.randn((1, H), generator=g, device=dev)
    steps = torch.arange(V, device=dev)[:, None] * (order / V) + 2.0
    w = (base * steps * 0.05).to(torch.bfloat16)
    x = (base + 0.02 * torch.randn((T, H), generator=g, device=dev)).to(torch.bfloat16)
    check_head(w, x, torch.arange(T, dtype=torch.int32, device=dev), 20)


def test_offsets_past_32_bits(dev):
    """More than 2^31 logits, and a head of more than 2^31 values."""
    from moe_offload_b200.tokens import head_logprobs, token_logprobs
    V, T = 248320, 8700
    lg = torch.zeros((T, V), device=dev)
    lg[T - 1, V - 1], lg[T - 1, 5], lg[T - 2, 7] = 9.0, 8.0, 7.0
    tg = torch.zeros(T, dtype=torch.int32, device=dev)
    tg[T - 1] = V - 1
    r = token_logprobs(lg, tg, 2)
    assert r.top_ids[T - 1].tolist() == [V - 1, 5] and r.top_ids[T - 2].tolist() == [7, 0]
    rest = math.log1p(math.exp(-1.0) + (V - 2) * math.exp(-9.0))
    assert abs(float(r.logprob[T - 1]) + rest) < RTOL * rest
    assert abs(float(r.logprob[0]) + math.log(V)) < 5e-4
    del lg
    V, H = 1_050_000, 2048
    w = torch.zeros((V, H), dtype=torch.bfloat16, device=dev)
    w[V - 1, 0], w[V - 2, 1], w[3, 2] = 4.0, 3.0, 2.0
    x = torch.ones((2, H), dtype=torch.bfloat16, device=dev)
    r = head_logprobs(w, x, torch.tensor([V - 1, V - 2], dtype=torch.int32, device=dev), 3)
    assert r.top_ids.tolist() == [[V - 1, V - 2, 3]] * 2
    lse = math.log(math.exp(4.0) + math.exp(3.0) + math.exp(2.0) + V - 3)
    assert abs(float(r.logprob[0]) - (4.0 - lse)) < HEAD_TOL * lse
    assert abs(float(r.logprob[1]) - (3.0 - lse)) < HEAD_TOL * lse


def test_refusals(dev):
    from moe_offload_b200.tokens import head_logprobs, token_logprobs
    lg = torch.zeros((2, 64), device=dev)
    tg = torch.zeros(2, dtype=torch.int32, device=dev)
    for bad in (lambda: token_logprobs(lg, tg, 33), lambda: token_logprobs(lg, tg, -1),
                lambda: token_logprobs(lg[:, :10].contiguous(), tg, 11), lambda: token_logprobs(lg[:, ::2], tg, 1),
                lambda: token_logprobs(lg.double(), tg, 1), lambda: token_logprobs(lg, tg.long(), 1),
                lambda: token_logprobs(lg, tg[:1], 1), lambda: token_logprobs(lg[0], tg, 1),
                lambda: token_logprobs(lg.cpu(), tg, 1)):
        with pytest.raises(ValueError):
            bad()
    w, x = torch.zeros((40, 64), dtype=torch.bfloat16, device=dev), torch.zeros((2, 64), dtype=torch.bfloat16, device=dev)
    for bad in (lambda: head_logprobs(w, x[:, :32].contiguous(), tg, 1), lambda: head_logprobs(w, x.float(), tg, 1),
                lambda: head_logprobs(w, x, tg, 41), lambda: head_logprobs(w, x, tg[:1], 1)):
        with pytest.raises(ValueError):
            bad()
