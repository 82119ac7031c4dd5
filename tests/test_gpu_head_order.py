"""Prompt scoring's order of the alternatives is that of the 64-bit logits where the tensor cores' sums say
otherwise: an entry whose large products cancel, beside leaders that they sum exactly.

The leaders are 10 + k * 2^-19 (k = 1 .. 60): two products in one step of 16, exact in fp32 (steps of 2^-20
from 8 on). The other entry is 20, then (H - 32) products of 2^-25, then -10 in the last step: beside 20 an
fp32 sum has steps of 2^-19, and each accumulation adds 16 * 2^-25 = 2^-21 < 2^-20 to it, which rounding to
nearest or towards zero drops. So the tensor cores see 10, below all leaders, where the sum is
10 + (H - 32) * 2^-25: for H = 4,096 62 leaders' steps, above all of them. Its magnitudes sum to 30, three times
the leaders' 10. For the statistics it is off by 1.2e-4 at one of 61 equal weights: 2e-6 of a log-probability of
-4, inside HEAD_TOL (relative, 1e-4)."""
import pytest
import torch

from test_gpu_logprobs import check_head

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch.device("cuda:0")


def cancelling(V, H, at):
    w, x = torch.zeros((V, H)), torch.zeros(H)
    x[0], x[1], x[H - 1] = 1.0, 2.0 ** -19, 1.0
    x[16:H - 16] = 2.0 ** -12
    w[:60, 0] = 10.0
    w[:60, 1] = torch.arange(1, 61).float()
    w[at, 0], w[at, H - 1] = 20.0, -10.0
    w[at, 16:H - 16] = 2.0 ** -13
    return w.bfloat16(), x.bfloat16()


@pytest.mark.parametrize("n", [1, 20, 32])
@pytest.mark.parametrize("T,V,at", [(1, 400, 300), (5, 30000, 29999), (140, 3000, 100), (600, 400, 399)])
def test_a_cancelling_entry_among_exact_leaders(dev, T, V, at, n):
    w, x = cancelling(V, 4096, at)
    x = x[None].repeat(T, 1).to(dev)
    r = check_head(w.to(dev), x, torch.full((T,), at, dtype=torch.int32, device=dev), n)
    assert r.top_ids[:, 0].tolist() == [at] * T


def test_equal_rows_of_zeros_need_no_second_look(dev):
    """Nothing is lost where there are no magnitudes: the ids in order, the log of V exactly."""
    w = torch.randn((5000, 64), device=dev).bfloat16()
    check_head(w, torch.zeros((3, 64), dtype=torch.bfloat16, device=dev), torch.tensor([0, 7, 4999], dtype=torch.int32,
                                                                                       device=dev), 20)
