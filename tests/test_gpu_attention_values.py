"""GPU tests of attention at the ends of the numbers: keys and values that are none, scores beyond
FP32, powers and queries far apart, in both kernels over the cache (up to 16 rows of queries to a
key head, and more)."""
import importlib
import math

import pytest
import torch

from test_gpu_attention import _filled, _int, _normal, _offsets

pytestmark = pytest.mark.gpu

D = 128


@pytest.fixture(scope="module")
def attention(package):
    return importlib.import_module("nemotron_inference_b200.attention")


@pytest.mark.parametrize("heads", [4, 32])
@pytest.mark.parametrize("half", [0, 1])
def test_no_number_far_below_the_largest_score(attention, heads, half):
    # the sequence is cut between blocks; the key or value stands in a first piece whose weights are all 2^-500
    # of those of the pieces that are joined with it: the formula multiplies by it all the same
    n = 20000
    cache = _filled(attention, [n, 30], 1, 64, seed=31, layers=1)
    pages = cache.block_table[0, :-(-n // 64)].long()
    codes = cache.codes.view(torch.uint8)
    low, high = (int(torch.tensor(x).to(torch.float8_e4m3fn).view(torch.uint8)) for x in (-16.0, 16.0))
    codes[0, pages, 0] = high
    codes[0, pages[:4], 0] = low
    cache.exponents[0, pages] = 0
    q = torch.ones((2, heads, D), dtype=torch.bfloat16, device="cuda")
    batch = (_int([0, 1]), _offsets([1, 1]))
    clean = cache.attend(0, q, *batch, scale=0.1)
    assert bool(clean.isfinite().all())
    codes[0, pages[1], half, 0, 40, 9] = 0x7F
    got = cache.attend(0, q, *batch, scale=0.1)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[0, :, slice(None) if half == 0 else 9] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool(got[hit].float().isnan().all())
    assert cache.sync_status() == 0


def _lowest(attention, lowest, of_even, check):
    # keys that are masked by a large negative value in a dimension of its own, which rows of even places
    # read; those of odd ones read another, and raise their references with the second tile
    n = 420
    k, v = (_normal(33 + i, n, 1, D) for i in range(2))
    q = _normal(35, n, 2, D)
    q[:, :, :2], k[:, :, :2] = 0, 0
    k[:256, 0, 0] = lowest
    k[128:256, 0, 1] = 100.0
    q[0::2, :, 0] = of_even
    q[1::2, :, 1] = 10.0
    q, k, v = (t.to(torch.bfloat16) for t in (q, k, v))
    got, lse = attention.attention_prefill(q, k, v, _offsets([n]), return_lse=True)
    assert attention.prefill_sync_status() == 0
    for h in range(2):
        scores = (q[:, h].double() @ k[:, 0].double().T) * D ** -0.5
        scores.masked_fill_(~torch.ones((n, n), dtype=torch.bool, device="cuda").tril(), -math.inf)
        # (by the maximum: a logarithm of the sum is lost beside a score of 1e30, in 64 bits as well)
        w = torch.exp(scores - scores.amax(1, keepdim=True))
        total = w.sum(1, keepdim=True)
        want, spread = (w @ v[:, 0].double()) / total, (w @ v[:, 0].double().abs()) / total
        bound = 1.75 * 2 ** -8 * spread + 2 ** -22 * v[:, 0].double().abs().sum(0) / total
        error = (got[:, h].double() - want).abs()
        assert bool((error <= bound)[check].all()), float((error / bound)[check].max())
        sums = scores.amax(1) + total[:, 0].log()
        off = (lse[:, h].double() - sums).abs() / sums.abs().clamp(min=64)
        assert float(off[check].max()) <= 2 ** -17


def test_prefill_of_rows_whose_first_scores_are_infinite(attention):
    # FP32 has no such number: -infinity, and those that a row sees later are finite
    _lowest(attention, -3.3895e38, 2.0, slice(256, None))


@pytest.mark.parametrize("lowest", [-1e4, -1e6, -1e9, -1e12, -1e30, -3.3895e38])
def test_prefill_of_scores_very_far_below_zero(attention, lowest):
    # the rows up to 256 see nothing else; between, FP32 holds such a sum's other terms in part
    _lowest(attention, lowest, 0.5, slice(256 if -1e30 < lowest < -1e4 else 0, None))
