"""Low-rank adapters beside a shared projection (moe_adapter_add) against the definition in 64 bits.

Tolerances. d = scale * sum_j u_j b_j with u_j = sum_k x_k a_k, both summed in fp32. The sum over K
is off by at most sqrt(K) * 2^-24 * sum|x a| for random signs (K * 2^-24 in the worst case), the sum
over the rank by rank * 2^-24 of sum|u b|, and u is carried with at least 2^-17 relative. In terms of
S = scale * sum_j (sum_k |x_k a_jk|) |b_j|, |d error| <= (K + rank) * 2^-24 S + 2^-17 S
<= 2e-4 S for K = 3072 + 128 in the worst case; random signs leave a tenth of it, which is asserted: 2e-5 S.
The result is rounded once: half a step of its type, 2^-8 of a bf16 value and 2^-24 of an fp32 one."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch.device("cuda:0")


def make(dev, T, K, N, r, banks, dtype, seed, ids=None):
    from moe_offload_b200.adapters import AdapterBank
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    bank = AdapterBank.synthetic(banks, r, K, N, dev, seed=seed + 1)
    bank.scale.copy_(torch.rand((banks,), generator=g, device=dev) * 2 - 0.5)
    x = torch.randn((T, K), generator=g, device=dev).to(torch.bfloat16)
    y = torch.randn((T, N), generator=g, device=dev).to(dtype)
    if ids is None:
        ids = torch.randint(-1, banks, (T,), generator=g, device=dev, dtype=torch.int32)
    else:
        ids = torch.tensor(ids, dtype=torch.int32, device=dev)
    return bank, x, y, ids


def check(bank, x, y, ids, out):
    want, size = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    for k in ids.unique().tolist():
        if not 0 <= k < bank.adapters:
            continue
        rows = (ids == k).nonzero()[:, 0]
        a, b, s = bank.a[k].double(), bank.b[k].double(), float(bank.scale[k])
        want[rows] += s * ((x[rows].double() @ a.t()) @ b.t())
        size[rows] = abs(s) * ((x[rows].double().abs() @ a.abs().t()) @ b.abs().t())
    half = 2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -24
    off = (out.double() - want).abs()
    bound = half * want.abs() + 2e-5 * size * (1 + half)
    assert bool((off <= bound).all()), float((off - bound).max())
    kept = ((ids < 0) | (ids >= bank.adapters)).nonzero()[:, 0]
    assert torch.equal(out[kept], y[kept])


SHAPES = [(1, 8, 1, 8, 1), (1, 2048, 768, 8, 4), (2, 64, 7, 16, 3), (3, 72, 100, 24, 2), (16, 256, 256, 32, 5),
          (17, 264, 257, 40, 5), (31, 1000, 333, 64, 3), (33, 3072, 768, 16, 40), (64, 768, 1000, 128, 9),
          (65, 520, 65, 120, 4), (100, 128, 4097, 8, 7), (300, 96, 130, 48, 300), (513, 768, 96, 16, 2),
          (40, 8, 8, 8, 1100), (9001, 16, 24, 8, 37), (2500, 64, 40, 32, 900), (2, 4096, 20000, 64, 2),
          # tiles of several rows: more than 74 rows and 32 MB of A and B, counted once for each row
          (75, 3072, 2048, 128, 11), (100, 3072, 2001, 64, 7), (130, 2048, 1030, 128, 5), (300, 1024, 1000, 64, 9),
          (300, 3080, 768, 16, 20), (700, 2056, 777, 8, 3), (1100, 1000, 1003, 56, 2), (1500, 768, 513, 24, 37),
          (2500, 512, 300, 16, 900), (2500, 264, 300, 40, 1100), (9001, 64, 72, 32, 37), (4100, 128, 33, 104, 50)]


@pytest.mark.parametrize("T,K,N,r,banks", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_against_definition(dev, T, K, N, r, banks, dtype):
    bank, x, y, ids = make(dev, T, K, N, r, banks, dtype, T + K + N)
    out = bank.add(y, x, ids)
    check(bank, x, y, ids, out)


@pytest.mark.parametrize("pattern", ["one", "none", "alternating", "runs", "last only", "each its own", "descending",
                                     "two thirds none"])
@pytest.mark.parametrize("T,K,N,r", [(1, 384, 200, 16), (15, 384, 200, 16), (16, 384, 200, 16), (48, 384, 200, 16),
                                     (130, 384, 200, 16), (77, 3072, 1024, 64), (130, 3072, 1024, 64),
                                     (600, 2048, 520, 16), (2049, 256, 256, 32), (5000, 64, 64, 32)])
def test_row_patterns(dev, pattern, T, K, N, r):
    banks = 7
    ids = {"one": [3] * T, "none": [-1] * T, "alternating": [t % 2 for t in range(T)],
           "runs": [t * 5 // T for t in range(T)], "last only": [-1] * (T - 1) + [6],
           "each its own": [t % banks for t in range(T)], "descending": [banks - 1 - t * banks // T for t in range(T)],
           "two thirds none": [t % banks if t % 3 == 0 else -1 for t in range(T)]}
    bank, x, y, ids = make(dev, T, K, N, r, banks, torch.bfloat16, T, ids[pattern])
    check(bank, x, y, ids, bank.add(y, x, ids))


def test_head_sized_projection(dev):
    bank, x, y, ids = make(dev, 4, 1024, 248320, 16, 3, torch.float32, 5, [2, -1, 0, 2])
    check(bank, x, y, ids, bank.add(y, x, ids))


def test_offsets_past_32_bits(dev):
    """More than 2^31 outputs, and a bank of more than 2^31 values."""
    from moe_offload_b200.adapters import AdapterBank
    T, N = 8700, 248320
    bank = AdapterBank.synthetic(2, 8, 8, N, dev)
    x = torch.ones((T, 8), dtype=torch.bfloat16, device=dev)
    y = torch.zeros((T, N), dtype=torch.float32, device=dev)
    ids = torch.full((T,), -1, dtype=torch.int32, device=dev)
    ids[T - 1], ids[0] = 1, 0
    out = bank.add(y, x, ids, out=y)
    rows = torch.tensor([0, T - 2, T - 1], device=dev)
    check(bank, x[rows], torch.zeros((3, N), dtype=torch.float32, device=dev), ids[rows], out[rows])
    del y, out
    bank = AdapterBank(torch.zeros((70, 128, 64), dtype=torch.bfloat16, device=dev),
                       torch.zeros((70, 248320, 128), dtype=torch.bfloat16, device=dev),
                       torch.ones(70, dtype=torch.float32, device=dev))
    bank.a[69] = 0.25
    bank.b[69, -5:] = 0.5
    x = torch.ones((3, 64), dtype=torch.bfloat16, device=dev)
    y = torch.zeros((3, 248320), dtype=torch.float32, device=dev)
    out = bank.add(y, x, torch.tensor([69, 68, -1], dtype=torch.int32, device=dev))
    assert bool((out[0, -5:] == 1024.0).all()) and not bool(out[0, :-5].any()) and not bool(out[1:].any())


@pytest.mark.parametrize("T,K,r", [(50, 256, 16), (150, 3072, 64)])
def test_in_place_and_out(dev, T, K, r):
    bank, x, y, ids = make(dev, T, K, 301, r, 4, torch.bfloat16, 6)
    want = bank.add(y, x, ids)
    buf = torch.full((T + 2, 301), 7.0, dtype=torch.bfloat16, device=dev)
    out = bank.add(y, x, ids, out=buf[1:T + 1])
    assert out.data_ptr() == buf[1:].data_ptr() and torch.equal(out, want)
    assert bool((buf[0] == 7).all()) and bool((buf[T + 1] == 7).all())    # nothing written around it
    keep = y.clone()
    assert bank.add(keep, x, ids, out=keep) is keep and torch.equal(keep, want)


@pytest.mark.parametrize("T,K,N,r", [(20, 64, 50, 8), (200, 3072, 1024, 64)])
def test_bad_ids_flagged_rows_kept(dev, T, K, N, r):
    from moe_offload_b200 import _lib
    bank, x, y, ids = make(dev, T, K, N, r, 3, torch.float32, 7, [0, 1, 2, 3, -2] + [-1] * (T - 10) + [1] * 5)
    _lib.call("moe_device_error", 1)
    out = bank.add(y, x, ids)
    torch.cuda.synchronize()
    assert int(_lib.call("moe_device_error", 1)) & 2
    check(bank, x, y, ids, out)
    bank.add(y, x, ids.clamp(max=2, min=-1))
    torch.cuda.synchronize()
    assert int(_lib.call("moe_device_error", 1)) == 0


@pytest.mark.parametrize("T,K,N,r", [(40, 128, 96, 16), (120, 3072, 1024, 64)])
def test_infinities_stay_in_their_rows(dev, T, K, N, r):
    """A row or an adapter with an inf or NaN changes no row that does not use it."""
    bank, x, y, ids = make(dev, T, K, N, r, 4, torch.float32, 8, [t % 4 for t in range(T)])
    want = bank.add(y, x, ids)
    x[5, 3] = float("inf")
    x[9, 0] = float("nan")
    bank.a[2, 0, 0] = float("nan")
    got = bank.add(y, x, ids)
    hit = (ids == 2) | (torch.arange(T, device=dev) == 5) | (torch.arange(T, device=dev) == 9)
    assert torch.equal(got[~hit], want[~hit])
    assert not bool(torch.isfinite(got[hit]).all(dim=1).any())


@pytest.mark.parametrize("T,K,r", [(70, 512, 32), (170, 3072, 64)])
def test_streams_and_graphs(dev, T, K, r):
    bank, x, y, ids = make(dev, T, K, 130, r, 6, torch.bfloat16, 9)
    want = bank.add(y, x, ids)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    side = bank.add(y, x, ids, stream=s)
    s.synchronize()
    assert torch.equal(side, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bank.add(y, x, ids)
    ids.copy_(ids.flip(0))                                   # the ids are read when the graph runs
    graph.replay()
    assert torch.equal(out, bank.add(y, x, ids))


def test_adapter_linear_beside_affine_projection(dev):
    from moe_offload_b200 import ops
    from moe_offload_b200.adapters import AdapterBank, adapter_linear
    from moe_offload_b200.synthetic import np_qmatrix, to_device_qmatrix
    rng = np.random.default_rng(10)
    K, N, T = 512, 192, 21
    w = to_device_qmatrix(np_qmatrix(rng, 1, N, K), dev)
    w = ops.QMatrix(w.w[0], w.s[0], w.b[0], w.bits, w.group_size)
    bank = AdapterBank.synthetic(3, 16, K, N, dev)
    x = torch.randn((T, K), device=dev).to(torch.bfloat16)
    ids = torch.tensor([t % 4 - 1 for t in range(T)], dtype=torch.int32, device=dev)
    y = adapter_linear(x, w, bank, ids)
    base = ops.affine_linear(x, w)
    check(bank, x, base, ids, y)
    assert torch.equal(y[0], base[0])


def test_empty_batch_and_refusals(dev):
    from moe_offload_b200._lib import MoeError
    from moe_offload_b200.adapters import AdapterBank
    bank, x, y, ids = make(dev, 4, 64, 64, 8, 2, torch.bfloat16, 11)
    assert bank.add(y[:0], x[:0], ids[:0]).shape == (0, 64)
    for bad in (lambda: bank.add(y.half(), x, ids), lambda: bank.add(y, x.float(), ids), lambda: bank.add(y, x, ids.long()),
                lambda: bank.add(y[:3], x, ids), lambda: bank.add(y, x[:, :56].contiguous(), ids),
                lambda: bank.add(y, x, ids[:3]), lambda: bank.add(y, x, ids, out=y.float()),
                lambda: bank.add(y.t(), x, ids), lambda: bank.add(y.cpu(), x, ids),
                lambda: AdapterBank(bank.a[:, :4].contiguous(), bank.b[:, :, :4].contiguous(), bank.scale),
                lambda: AdapterBank(bank.a, bank.b[:1], bank.scale), lambda: AdapterBank(bank.a, bank.b, bank.scale[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(MoeError):
        bank.add(y, x, ids, out=x)                           # out over another input
    wide = torch.zeros((9, 64), dtype=torch.bfloat16, device=dev)
    with pytest.raises(MoeError):
        bank.add(wide[:4], x, ids, out=wide[1:5])            # out over a part of y


@pytest.mark.parametrize("rank", [8, 16, 24, 40, 72])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [2, 2000])
def test_infinite_inputs_stay_infinite(rank, dtype, T):
    """An infinity in x with a and b positive: the row's outputs are +inf by the formula, and no NaN comes from
    places behind the rank. Two rows go one a tile, 2,000 in tiles of several; the other rows stay finite."""
    from moe_offload_b200.adapters import AdapterBank
    dev = torch.device("cuda:0")
    K = N = 1024
    bank = AdapterBank(torch.full((2, rank, K), 0.01, dtype=torch.bfloat16, device=dev),
                       torch.full((2, N, rank), 0.5, dtype=torch.bfloat16, device=dev),
                       torch.ones(2, device=dev))
    x = torch.ones((T, K), dtype=torch.bfloat16, device=dev)
    x[1, 3] = float("inf")
    y = torch.zeros((T, N), dtype=dtype, device=dev)
    out = bank.add(y, x, (torch.arange(T, device=dev) % 2).int())
    assert torch.isposinf(out[1]).all()
    assert torch.isfinite(out[torch.arange(T, device=dev) != 1]).all()
