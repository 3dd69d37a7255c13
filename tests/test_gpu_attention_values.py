"""GPU tests of attention at the ends of the numbers: keys and values that are none, scores beyond
FP32, powers and queries far apart, in both kernels over the cache (up to 16 rows of queries to a
key head, and more).

Tolerances, per element, with A the softmax-weighted sum of |v| behind it:
- results are bf16, off by half a unit in the last place: 2^-8 of the value at most (just above a
  power of two), which A bounds;
- weights enter the second product as bf16 or as two E4M3 terms: 2^-8 of each at most, 2^-8 A.  The
  E4M3 terms end at 2^-22, where the largest weight of a row is 2^-1.5 at least: 2^-20.5 of that, a
  token each;
- scores are FP32 sums and the exponentials good to 2^-13: 2^-10 A for scores within 64.  Over the
  cache a query is two E4M3 terms with the row's largest element between 2^7 and 2^8, and the
  second is rounded to 2^-10 at worst in the kernel for many rows: 2^-17 of the largest in each element,
  delta = scale 2^-17 max|q| sum|k| in a score.  That changes a weight by a factor e^(+-delta) and
  the result by 2 delta A to first order (2.2 here: delta < 0.1).
Together (2.25 2^-8 + 2.2 delta) A + 2^-20.5 w_max sum|v|."""
import importlib
import math

import pytest
import torch

from test_gpu_attention import _check_attend, _filled, _int, _normal, _offsets, _values

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
        want, bound = (w @ v[:, 0].double()) / total, _bound(w / total, v[:, 0].double())
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


def _bound(w, v, delta=0.0):
    """w [rows, tokens], v [tokens, D]."""
    return (2.25 * 2 ** -8 + 2.2 * delta) * (w @ v.abs()) + 2 ** -20.5 * w.amax(1, keepdim=True) * v.abs().sum(0)


# 32 query heads to a key head: more than 16 rows of queries in every entry
@pytest.mark.parametrize("heads,kv_heads", [(32, 1), (64, 2)])
@pytest.mark.parametrize("length", [133, 9000])
def test_many_rows_keep_what_is_masked_out(attention, heads, kv_heads, length):
    rows, other, at = 6, 2, length - 3  # row 3 and later ones see the token
    cache = _filled(attention, [length, 70], kv_heads, 64, seed=5, layers=1)
    group, head = heads // kv_heads, kv_heads - 1
    q = _normal(13, rows + other, heads, D).to(torch.bfloat16)
    batch = (_int([0, 1]), _offsets([rows, other]))
    clean = cache.attend(0, q, *batch)
    bits = cache.codes.view(torch.uint8)
    page = int(cache.block_table[0, at // 64])
    for half in (0, 1):
        place = (0, page, half, head, at % 64, 9)
        before = int(bits[place])
        bits[place] = 0xFF if half else 0x7F
        got = cache.attend(0, q, *batch)
        bits[place] = before
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[3:rows, head * group:(head + 1) * group, 9 if half else slice(None)] = True
        assert torch.equal(got[~hit], clean[~hit]) and bool(got[hit].float().isnan().all())
    assert torch.equal(cache.attend(0, q, *batch), clean) and cache.sync_status() == 0


@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("heads,counts", [(32, [3, 1]), (128, [1, 1])])
def test_many_rows_over_pages_of_very_different_scales(attention, page_tokens, heads, counts):
    n = 4000
    cache = _filled(attention, [n, 90], 1, page_tokens, seed=3, layers=1)
    pages = cache.block_table[0, :-(-n // page_tokens)].long()
    # values up to 2^64 apart; the largest keys stand where the values are small
    g = torch.Generator().manual_seed(4)
    big = torch.rand(pages.numel(), generator=g) < 0.3
    powers = torch.randint(-32, 33, (pages.numel(),), generator=g)
    cache.exponents[0, pages, 1, 0] = torch.where(big, -32, powers).to(torch.int8).cuda()
    cache.exponents[0, pages, 0, 0] = torch.where(big, -5, torch.randint(-32, -6, (pages.numel(),), generator=g)).to(
        torch.int8).cuda()
    q = _normal(11, sum(counts), heads, D).to(torch.bfloat16)
    got = cache.attend(0, q, _int([0, 1]), _offsets(counts))
    _check_attend(cache, 0, q, [0, 1], counts, got)


def _check_many_rows(cache, q, scale, got):
    """One row of 32 or more heads of sequence 0."""
    k, v = _values(cache, 0, 0)
    group = q.shape[1] // cache.kv_heads
    for h in range(q.shape[1]):
        x = q[0, h].double()
        delta = scale * 2 ** -17 * float(x.abs().max()) * float(k[h // group].abs().sum(1).max())
        assert delta < 0.1
        w = torch.softmax((k[h // group] @ x) * scale, 0)[None]
        bound = _bound(w, v[h // group], delta)
        error = (got[0, h].double() - w @ v[h // group]).abs()
        assert bool((error <= bound).all()), (h, float((error / bound).max()))


def test_many_rows_of_queries_of_any_size(attention):
    # rows whose elements lie many powers of two apart, rows of zeros, rows near bf16's ends, outliers
    heads = 64
    cache = _filled(attention, [300, 300], 2, 32, seed=4, layers=1)
    q = _normal(12, 6, heads, D)
    q[0] *= torch.exp2(torch.linspace(-30, 0, D, device="cuda"))
    q[1] = 0
    q[2] *= 2.0 ** -100
    q[3] *= 2.0 ** 20
    q[4, :, 5] = 2.0 ** 9
    q[5, :, 5] = torch.exp2(torch.arange(heads, device="cuda") / 8.0 + 2)
    q = q.to(torch.bfloat16)
    pages = cache.block_table[0, :10].long()
    for row, scale in ((0, 0.1), (1, 0.1), (2, 0.1), (2, 2.0 ** 97), (3, 2.0 ** -23), (4, 0.01), (5, 0.01)):
        if row >= 4:  # (the outlier meets keys of nothing: what is left depends on the other elements)
            cache.codes.view(torch.uint8)[0, pages, 0, :, :, 5] = 0
        got = cache.attend(0, q[row:row + 1], _int([0]), _offsets([1]), scale=scale)
        _check_many_rows(cache, q[row:row + 1], scale, got)
    assert cache.sync_status() == 0


@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("power", [4, 14, 24, 32])
def test_scores_far_above_those_of_the_tiles_before(attention, heads, power):
    # the first 192 tokens are masked by keys that are lowest in one dimension: their scores are -448 x 2^power
    # x scale, and the tokens behind them alone count.  Blocks have several tiles of a sequence each.
    n, kv_heads, masked, scale = 700, 4, 192, D ** -0.5
    cache = _filled(attention, [n] * 40, kv_heads, 64, seed=41, layers=1)
    codes = cache.codes.view(torch.uint8)
    codes[0, :, 0, :, :, 0] = 0
    pages = cache.block_table[:, :masked // 64].flatten().long()
    codes[0, pages, 0] = 0
    codes[0, pages, 0, :, :, 0] = 0xFE  # -448
    cache.exponents[0, pages, 0] = power
    q = _normal(42, 40, heads, D)
    q[:, :, 0] = 1.0
    q = q.to(torch.bfloat16)
    everyone = list(range(40))
    got = cache.attend(0, q, _int(everyone), _offsets([1] * 40))
    assert cache.sync_status() == 0
    group = heads // kv_heads
    for s in everyone:
        k, v = _values(cache, 0, s)
        for h in range(kv_heads):
            of = slice(h * group, (h + 1) * group)
            x = q[s, of].double()
            scores = (x @ k[h].T) * scale
            w = torch.softmax(scores, 1)
            # (of the tokens that count)
            bound = _bound(w, v[h], scale * 2 ** -17 * float(x.abs().max()) * float(k[h, masked:].abs().sum(1).max()))
            error = (got[s, of].double() - w @ v[h]).abs()
            assert bool((error <= bound).all()), (s, h, float((error / bound).max()))
