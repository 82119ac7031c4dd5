"""Log-probabilities of rows whose logits all lie far below 0, where threads or warps of the row hold
nothing at all (rows shorter than a CTA, masks that leave little): the definition's results, at the
tolerances derived in test_gpu_logprobs. A shift moves every logit alike, so it changes the rounding
of the inputs only, which both sides see."""
import numpy as np
import pytest
import torch

from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch.device("cuda:0")


def low_rows(T, V, shift, masked, rng):
    """N(0, 3) + shift; a part of them masked, never the whole row."""
    lg = (rng.normal(0, 3, (T, V)) + shift).astype(np.float32)
    if masked:
        gone = rng.random((T, V)) < masked
        gone[np.arange(T), rng.integers(0, V, T)] = False
        lg[gone] = -np.inf
    return lg


@pytest.mark.parametrize("shift", [-100.0, -1e4, -3e38])
@pytest.mark.parametrize("masked", [0.0, 0.5, 0.99])
@pytest.mark.parametrize("T,V", [(1, 1), (2, 5), (3, 257), (2, 1000), (2, 9001), (3, 50021), (1, 248320),
                                 (160, 257), (300, 20001)])
def test_low_rows(dev, T, V, masked, shift):
    rng = np.random.default_rng(V + int(100 * masked))
    lg = low_rows(T, V, shift, masked, rng)
    check(lg, rng.integers(0, V, T), min(V, 20), dev)


@pytest.mark.parametrize("V", [1, 5, 257, 1000, 50021])
def test_rows_of_the_lowest_value(dev, V):
    """The type's lowest value everywhere (a uniform row), and beside masked entries."""
    low = np.finfo(np.float32).min
    lg = np.full((2, V), low, np.float32)
    lg[1, : V // 2] = -np.inf
    check(lg, [0, V - 1], min(V, 32), dev)


def test_nan_in_a_row_without_anything_else(dev):
    """What a thread without a finite logit passes on: a NaN, also where others hold low logits."""
    lg = np.full((3, 257), -np.inf, np.float32)
    lg[0, 256] = -500.0
    lg[1, 256], lg[1, 3] = -500.0, np.nan
    lg[2, 3] = np.nan
    check(lg, [256, 256, 0], 5, dev)


def test_decode_of_low_logits(dev):
    """A uniform row at -100: log(V), whatever the size."""
    from moe_offload_b200.tokens import token_logprobs
    for V in (3, 257, 1024):
        r = token_logprobs(torch.full((1, V), -100.0, device=dev), torch.zeros(1, dtype=torch.int32, device=dev), 1)
        assert abs(float(r.logprob[0]) + np.log(V)) < 1e-5 and abs(float(r.entropy[0]) - np.log(V)) < 1e-5
