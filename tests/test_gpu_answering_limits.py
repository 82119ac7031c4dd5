"""Borders of the answering operators' precision and launch rules.

Sums of a row of logits: from 296 rows on, up to 131,072 logits go through 256 threads a row, 512 terms a
thread, one after another, then 5 merges in a warp and 8 warps' sums: 525 * 2^-24 = 3.1e-5 if all roundings
had one sign, beside the 30 * 2^-23 + 2^-22 of an exponential: below 4e-5, inside the RTOL of
test_gpu_logprobs (5e-5). Other launches add at most 485 terms (V / 512, or V / 256 and V / 128 up to V = 16,384).

Adapters' fp32 outputs: u = x . A^T goes into the second product as three bf16 numbers, which hold all of an fp32
number. Here u is a sum of three products of one step (a 24-bit number) and each output is one u, so that the
first product may lose 3 * 2^-23 (a truncation each) and the second as much in its three parts: 7.2e-7 of the
result. Two parts would leave up to 2^-17 = 7.6e-6."""
import numpy as np
import pytest
import torch

from test_gpu_logprobs import close, plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch.device("cuda:0")


@pytest.mark.parametrize("T,V", [(295, 131072), (296, 131072), (296, 131073), (148, 16384), (147, 16384)])
def test_longest_sums_of_the_launch_rules(dev, T, V):
    from moe_offload_b200.tokens import token_logprobs
    rng = np.random.default_rng(T + V)
    lg = rng.normal(0, 0.01, (3, V)).astype(np.float32)
    lg[1] = np.sort(lg[1])                                # (alike, so that roundings may go one way)
    lg[2] = 1.0
    targets = np.array([0, V - 1, 5])
    kind = torch.arange(T, device=dev) % 3
    r = token_logprobs(torch.from_numpy(lg).to(dev)[kind], torch.from_numpy(targets.astype(np.int32)).to(dev)[kind], 4)
    lp, en, ids, tl = plain(lg, targets, 4)
    assert np.array_equal(r.top_ids[:3].cpu().numpy(), ids)
    for got, want in ((r.logprob, lp), (r.entropy, en), (r.top_logprobs, tl)):
        close(got[:3], want, "first rows")
        assert torch.equal(got, got[:3][kind])


@pytest.mark.parametrize("T,K,N,rank", [(200, 768, 1024, 64), (150, 512, 1000, 128), (900, 768, 1026, 16), (2048, 256, 264, 24)])
def test_adapters_fp32_outputs_keep_all_bits_of_u(dev, T, K, N, rank):
    from moe_offload_b200.adapters import AdapterBank
    assert T > 74 and T * rank * (K + N) * 2 > 32e6       # the tensor cores' tiles
    g = torch.Generator().manual_seed(rank)
    a = torch.zeros((2, rank, K))
    bits = torch.randint(128, 256, (2, rank, 3), generator=g).float()
    a[:, :, :3] = bits / 128.0
    x = torch.zeros((T, K))
    x[:, 0], x[:, 1], x[:, 2] = 1.0, 2.0 ** -8, 2.0 ** -16
    b = torch.zeros((2, N, rank))
    of = torch.randint(0, rank, (2, N), generator=g)
    b.scatter_(2, of[:, :, None], 1.0)
    ids = torch.randint(0, 2, (T,), generator=g)
    u = (bits / 128.0).double() @ torch.tensor([1.0, 2.0 ** -8, 2.0 ** -16], dtype=torch.float64)
    want = torch.gather(u, 1, of)[ids]
    bank = AdapterBank(a.bfloat16().to(dev), b.bfloat16().to(dev), torch.ones(2, device=dev))
    got = bank.add(torch.zeros((T, N), device=dev), x.bfloat16().to(dev), ids.int().to(dev)).cpu().double()
    assert float(((got - want).abs() / want.abs()).max()) < 1e-6


def test_adapters_on_the_head_need_ids(dev):
    from moe_offload_b200.adapters import AdapterBank
    from moe_offload_b200.tokens import TokenHead
    head, bank = TokenHead.synthetic(300, 64, dev), AdapterBank.synthetic(2, 8, 64, 300, dev)
    h = torch.ones((2, 64), dtype=torch.bfloat16, device=dev)
    ids = torch.zeros(2, dtype=torch.int32, device=dev)
    out = torch.full((2, 300), 7.0, device=dev)
    with pytest.raises(ValueError, match="adapter_ids"):
        head.logits(h, out=out, adapters=bank)
    assert bool((out == 7.0).all())                       # refused before anything ran
    head.logits(h, out=out, adapters=bank, adapter_ids=ids)
