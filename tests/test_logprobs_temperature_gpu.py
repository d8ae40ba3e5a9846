"""csdr_token_logprobs at temperatures whose quotients leave fp32 or round to equals, against fp64
numpy."""
import numpy as np
import pytest

from test_logprobs_rounds_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [0.25, 0.7, 1.3, 0.9999999])
@pytest.mark.parametrize("copies", [1, 1366])  # (one round a segment, and all of them in one)
def test_masks_of_the_lowest_value(gpu, temperature, copies):
    """Rows of nothing but the lowest value are uniform; where fewer tokens are allowed than the top
    has places, masked ones follow in order of their ids."""
    n = 6000
    low = np.finfo(np.float32).min
    x = np.full((6, n), low, np.float32)
    rng = np.random.default_rng(5)
    x[1, ::1000] = rng.normal(size=6)
    x[2, :3000] = rng.normal(size=3000)
    x[3, 4096:] = -np.inf
    x[4, 5999] = -low
    x[5, 17] = low / 2
    check(gpu, x, [3, 1000, 3500, 5000, 5999, 17], 20, temperature, copies=copies)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("temperature", [1.2e-38, 1e-30, 1e-6, 1e6, 1e30])
def test_far_temperatures(gpu, dtype, temperature):
    """The smallest temperature leaves the likeliest token alone, the largest makes all alike; the
    order of the top is that of the logits."""
    x = (4 * np.random.default_rng(6).normal(size=(5, 5001))).astype(dtype)
    x[1, :2100] = 0.0
    x[2] = np.abs(x[2])
    x[3] = -np.abs(x[3])
    check(gpu, x, [int(x[0].argmax()), 2100, 1, 2, 3], 20, temperature)


@pytest.mark.parametrize("temperature", [0.7, 3.0, 1.9])
def test_neighbouring_logits(gpu, temperature):
    """Neighbouring fp32 values, some of whose quotients round to the same: ranked by the logits,
    ties only where these are equal."""
    x = (np.float32(1.6).view(np.int32) + np.arange(4000) // 2).astype(np.int32).view(np.float32)
    x = np.stack([x, x[::-1], -x])
    check(gpu, x, [3999, 0, 1], 64, temperature)
