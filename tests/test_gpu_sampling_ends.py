"""GPU tests of sampling where rounding decides: random numbers at the ends of rows of very light tokens, borders between
a sum and the sum of its rounded terms, and log-probabilities.

Tokens are the definition's.  Log-probabilities: x - m and the logarithm are FP64, the sum of e^(x - m) is within 2^-36 of
itself for its terms, 2^-40 for the order of adding, and what lies below 2^-64 of the largest (2^-64 131072 at most) is left
out: 2^-35 altogether, and the result is FP32: half a step, 2^-24 of it."""
import importlib
import math

import numpy as np
import pytest
import torch

from test_gpu_sampling import _logits, _token

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampling(package):
    return importlib.import_module("nemotron_inference_b200.sampling")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(8, 131072), (90, 50001), (3, 300), (8, 20000)])
@pytest.mark.parametrize("light", [-31.25, -31.75, -33.0])
def test_ends_of_rows_whose_first_or_last_tokens_weigh_next_to_nothing(sampling, light, rows, vocab, dtype):
    """Weights of 0.47, 0.29 and 0.08 2^-44 of the largest: each rounds to nothing, their sums do not."""
    assert math.exp(light) * 2 ** 44 < 0.5
    for place in (0, vocab // 2, vocab - 1):
        logits = torch.full((rows, vocab), light, device="cuda", dtype=dtype)
        logits[:, place] = 0.0
        for u, first in ((0.0, True), (1e-30, True), (-1.0, True), (math.nan, True), (1.0, False), (2.0, False), (math.inf, False)):
            uniform = torch.full((rows,), u, device="cuda")
            for setting in (dict(), dict(min_p=1e-20), dict(top_k=vocab - 1)):
                tokens, logprobs = sampling.sample(logits, uniform, return_logprobs=True, **setting)
                assert bool(((tokens >= 0) & (tokens < vocab)).all()), (place, u, setting)
                assert bool(logprobs.isfinite().all())
                if not setting and vocab > 1000 and light > -32.0:
                    # those of a thread, four or more, weigh a unit together: the row's first and last tokens count
                    end = 0 if first else vocab - 1
                    if place != end:
                        assert bool((tokens == end).all()), (place, u, tokens[:4])
                    else:
                        assert bool((tokens == place).all())


def _between_sums():
    """Logits of three values, and a top_p, for which the tokens that stay - the largest and all of the second value -
    reach p of the sum, but do not if each one's weight is rounded to 2^-44 of the largest first.  The third value is that of
    the tokens which the search guesses by."""
    vocab, unit = 131072, 2.0 ** 44
    sampled = np.arange(vocab) % 1024 < 64  # (for up to 13 rows: a sixteenth)
    n_third = int(sampled.sum())
    n_second = vocab - n_third - 1
    second = np.float32(-10.0)
    while not 0.38 < (math.exp(float(second)) * unit) % 1.0 < 0.42:
        second = np.nextafter(second, np.float32(0))
    of_second = math.exp(float(second)) * unit
    above = unit + n_second * of_second
    gap = n_second * (of_second % 1.0)
    third = np.float32(-11.5)
    while True:
        whole = above + n_third * math.exp(float(third)) * unit
        top_p = np.float32((above - gap / 2) / whole)
        if abs(float(top_p) * whole - (above - gap / 2)) < gap / 8:
            break
        third = np.nextafter(third, np.float32(0))
    x = np.where(sampled, third, second).astype(np.float32)
    x[100] = 0.0  # (not one of the guess's)
    return x, float(top_p)


def test_a_border_between_a_sum_and_that_of_its_rounded_terms(sampling):
    x, top_p = _between_sums()
    uniform = np.linspace(0.05, 0.95, 8).astype(np.float32)
    logits = torch.from_numpy(x)[None].repeat(8, 1).cuda()
    tokens = sampling.sample(logits, torch.from_numpy(uniform).cuda(), top_p=top_p).tolist()
    assert all(x[token] > x.min() for token in tokens)
    assert tokens == [_token(x, u, top_p=top_p)[0] for u in uniform]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(2, 131072), (40, 1000), (80, 50001), (5, 33)])
def test_log_probabilities(sampling, rows, vocab, dtype):
    for number, spread in enumerate((0.5, 2.0, 8.0)):
        logits, uniform = _logits(rows, vocab, dtype, 60 + number, spread=spread)
        for setting in (dict(), dict(temperature=0.0), dict(temperature=0.7, top_p=0.9), dict(top_k=20)):
            tokens, logprobs = sampling.sample(logits, uniform, return_logprobs=True, **setting)
            x = logits.double()
            want = (x - torch.logsumexp(x, dim=1, keepdim=True)).gather(1, tokens[:, None].long())[:, 0]
            error = (logprobs.double() - want).abs()
            assert bool((error <= 2.0 ** -24 * want.abs() + 2.0 ** -34).all()), (setting, float(error.max()))
