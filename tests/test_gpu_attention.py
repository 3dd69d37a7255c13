"""GPU tests of the attention operators: prompts, the paged 8-bit cache, and its pages, each against
a plain implementation in 64 bits (or, for what moves pages, whole numbers in Python).

Tolerances, per element, with A the softmax-weighted sum of |v| behind it:
- results are bf16: 2^-9 of the value, which A bounds;
- the weights enter the second product rounded to bf16, or as two E4M3 terms: 2^-8 of each at most,
  2^-8 A together; the E4M3 terms also end at 2^-22 of the largest weight, a token each;
- scores are FP32 sums of 128 products, at most 2^-17 of sum |q k| off, and the exponentials are good
  to 2^-20: with scores within 64, below 2^-10 A.
Together 1.75 * 2^-8 A + 2^-22 w_max sum |v|."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


@pytest.fixture(scope="module")
def attention(package):
    return importlib.import_module("nemotron_inference_b200.attention")


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return _int(at)


def _normal(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def _rows(q, k, v, first, scale):
    """Row j of q [rows, D] sees the first + j + 1 first tokens of k, v [tokens, D] (64 bits)."""
    scores = (q @ k.T) * scale
    seen = torch.arange(k.shape[0], device="cuda")[None] <= \
        first + torch.arange(q.shape[0], device="cuda")[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(scores, dim=1)
    w = torch.exp(scores - lse[:, None])
    spread = w @ v.abs()
    bound = 1.75 * 2 ** -8 * spread + 2 ** -22 * w.amax(1, keepdim=True) * v.abs().sum(0)
    return w @ v, lse, bound


def _check_prefill(q, k, v, lengths, got, lse=None, scale=D ** -0.5):
    group = q.shape[1] // k.shape[1]
    start = 0
    for n in lengths:
        rows = slice(start, start + n)
        for h in range(q.shape[1] if n else 0):
            want, sums, bound = _rows(q[rows, h].double(), k[rows, h // group].double(),
                                      v[rows, h // group].double(), 0, scale)
            error = (got[rows, h].double() - want).abs()
            assert bool((error <= bound).all()), (n, h, float((error / bound).max()))
            if lse is not None:
                assert float((lse[rows, h].double() - sums).abs().max()) <= 2 ** -17 * 64
        start += n


@pytest.mark.parametrize("lengths", [[1], [2], [17], [128], [129], [257, 1], [1, 0, 127, 128, 5],
                                     [0, 300, 0], [600], [33] * 40])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 3), (5, 1), (16, 1)])
def test_prefill_against_64_bits(attention, lengths, heads, kv_heads):
    t = sum(lengths)
    x = _normal(t + heads, t, heads + 2 * kv_heads, D).to(torch.bfloat16)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    got, lse = attention.attention_prefill(q, k, v, _offsets(lengths), return_lse=True)
    assert attention.prefill_sync_status() == 0
    _check_prefill(q, k, v, lengths, got, lse)
    again = attention.attention_prefill(q, k, v, _offsets(lengths))
    assert torch.equal(again, got)  # the same bits every time, with or without the sums


@pytest.mark.parametrize("lengths,heads,kv_heads", [
    ([2100], 32, 2), ([700, 1300, 40, 0, 950], 16, 8), ([1500, 300], 15, 5), ([128] * 20, 40, 8)])
def test_prefill_with_more_tiles_than_blocks(attention, lengths, heads, kv_heads):
    t = sum(lengths)
    q, k, v = (_normal(50 + i, t, h, D).to(torch.bfloat16) for i, h in enumerate((heads, kv_heads, kv_heads)))
    got, lse = attention.attention_prefill(q, k, v, _offsets(lengths), return_lse=True)
    assert attention.prefill_sync_status() == 0
    _check_prefill(q, k, v, lengths, got, lse)
    for _ in range(3):
        assert torch.equal(attention.attention_prefill(q, k, v, _offsets(lengths)), got)
    assert attention.prefill_sync_status() == 0


def test_prefill_of_separate_tensors_and_a_scale_of_its_own(attention):
    n, heads, kv_heads = 321, 6, 2
    q = _normal(1, n, heads, D).to(torch.bfloat16)
    k = _normal(2, n, kv_heads + 1, D).to(torch.bfloat16)[:, 1:]
    v = _normal(3, n, kv_heads, D).to(torch.bfloat16)
    out = torch.full((n, heads, D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = attention.attention_prefill(q, k, v, _offsets([n]), scale=0.3, out=out)
    assert got is out
    _check_prefill(q, k, v, [n], got, scale=0.3)


def test_prefill_of_scores_far_from_zero(attention):
    # row maxima that rise from tile to tile, and scores that all lie far below zero
    n, heads = 700, 2
    k = _normal(5, n, 1, D).to(torch.bfloat16)
    k[:, 0, 0] = torch.linspace(-8, 8, n, device="cuda").to(torch.bfloat16)
    q = (0.1 * _normal(6, n, heads, D)).to(torch.bfloat16)
    q[:, 0, 0], q[:, 1, 0] = 64.0, -64.0
    v = _normal(7, n, 1, D).to(torch.bfloat16)
    got = attention.attention_prefill(q, k, v, _offsets([n]))
    _check_prefill(q, k, v, [n], got)


@pytest.mark.parametrize("token", range(20, 29))
def test_prefill_of_a_key_that_is_no_number(attention, token):
    # wherever it stands in its tile: the rows that see it are no numbers, those before it are the same
    q, k, v = (_normal(40 + i, 150, h, D).to(torch.bfloat16) for i, h in enumerate((2, 1, 1)))
    clean = attention.attention_prefill(q, k, v, _offsets([150]))
    k[token, 0, 7] = math.nan
    got = attention.attention_prefill(q, k, v, _offsets([150]))
    assert torch.equal(got[:token], clean[:token]) and bool(got[token:].float().isnan().all())


@pytest.mark.parametrize("heads,token", [(2, t) for t in range(64, 74)] + [(32, t) for t in range(64, 74)])
def test_attend_to_a_key_that_is_no_number(attention, heads, token):
    cache = _filled(attention, [100, 100], 1, 64, seed=6, layers=1)
    q = _normal(14, 2, heads, D).to(torch.bfloat16)
    batch = (_int([0, 1]), _offsets([1, 1]))
    clean = cache.attend(0, q, *batch)
    page = int(cache.block_table[1, token // 64])
    cache.codes.view(torch.uint8)[0, page, 0, 0, token % 64, 11] = 0x7F
    got = cache.attend(0, q, *batch)
    assert torch.equal(got[0], clean[0]) and bool(got[1].float().isnan().all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prefill_keeps_what_is_masked_out(attention, bad):
    lengths, heads = [100, 260, 40], 4
    t = sum(lengths)
    q, k, v = (_normal(20 + i, t, h, D).to(torch.bfloat16) for i, h in enumerate((heads, 2, 2)))
    at, offsets = 100 + 150, _offsets(lengths)  # token 150 of the second prompt
    clean = attention.attention_prefill(q, k, v, offsets)
    v2 = v.clone()
    v2[at, 1, 5] = bad
    got = attention.attention_prefill(q, k, v2, offsets)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[at:360, 2:, 5] = True  # the rows that see it, in the heads and the column that read it
    assert torch.equal(got[~hit], clean[~hit])
    seen = got[hit].float()
    assert bool(seen.isnan().all() if math.isnan(bad) else (seen == bad).all())
    k2 = k.clone()
    k2[at, 0, 3] = math.nan
    got = attention.attention_prefill(q, k2, v, offsets)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[at:360, :2] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool(got[hit].float().isnan().all())


def test_prefill_on_another_stream_and_replayed_from_a_graph(attention):
    q, k, v = (_normal(30 + i, 200, h, D).to(torch.bfloat16) for i, h in enumerate((4, 2, 2)))
    offsets = _offsets([120, 80])
    out = torch.empty_like(q)
    want = attention.attention_prefill(q, k, v, offsets)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        attention.attention_prefill(q, k, v, offsets, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention.attention_prefill(q, k, v, offsets, out=out)
    offsets.copy_(_offsets([50, 150]))  # read when the graph runs
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, attention.attention_prefill(q, k, v, _offsets([50, 150])))


def test_prefill_refusals(attention, package):
    q, k = (torch.zeros((8, h, D), dtype=torch.bfloat16, device="cuda") for h in (4, 2))
    offsets = _offsets([8])
    for bad_q, bad_k, bad_offsets in [
            (q.float(), k, offsets), (q[..., :64], k, offsets), (q.cpu(), k, offsets),
            (q.transpose(0, 1), k, offsets), (q, k, offsets.long()), (q, k, offsets.cpu())]:
        with pytest.raises(ValueError):
            attention.attention_prefill(bad_q, bad_k, bad_k, bad_offsets)
    with pytest.raises(ValueError):
        attention.attention_prefill(q, k, k, offsets, out=torch.zeros_like(q).float())
    for bad_q, bad_k, bad_v, scale in [
            (q[:, :3], k, k, None), (q, k[:4], k[:4], None), (q, k, k[:4], None), (q, k, k, -1.0),
            (q, k, k, math.nan), (q, k, k, 0.0)]:
        with pytest.raises(package.NmoeError):
            attention.attention_prefill(bad_q, bad_k, bad_v, offsets, scale=scale)
    odd = torch.zeros(8 * 4 * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(8, 4, D)
    with pytest.raises(package.NmoeError):  # rows that do not begin on 16 bytes
        attention.attention_prefill(odd, k, k, offsets)
    assert attention.attention_prefill(q[:0], k[:0], k[:0], _offsets([0])).shape == (0, 4, D)


# ---------------------------------------------------------------------------
# The cache
# ---------------------------------------------------------------------------

def _filled(attention, lengths, kv_heads, page_tokens, seed, layers=2, spare=3):
    """A cache whose sequences hold `lengths` tokens in scattered pages.  Every place that no
    sequence has reached, and every free page, holds NaN codes."""
    held = [-(-n // page_tokens) for n in lengths]
    total = sum(held) + spare
    cache = attention.KvCache.allocate(layers, total, kv_heads, len(lengths), max(held + [1]) + 1,
                                       page_tokens)
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(total, generator=g)
    codes = (_normal(seed, *cache.codes.shape) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    reached = torch.zeros((total, page_tokens), dtype=torch.bool)
    at = 0
    for i, n in enumerate(lengths):
        pages = order[at:at + held[i]]
        cache.block_table[i, :held[i]] = pages.int().cuda()
        flat = torch.arange(held[i] * page_tokens) < n
        reached[pages] = flat.view(held[i], page_tokens)
        cache.references[pages.cuda()] = 1
        at += held[i]
    bits = codes.view(torch.uint8)
    bits.masked_fill_(~reached.cuda()[None, :, None, None, :, None], 0x7F)
    cache.codes.copy_(codes)
    cache.exponents.copy_(torch.randint(-9, -3, cache.exponents.shape, generator=g).to(torch.int8))
    cache.lengths.copy_(_int(lengths))
    return cache


def _values(cache, layer, sequence):
    """Keys and values [2, kv_heads, tokens, D] of a sequence, in 64 bits."""
    n, p = int(cache.lengths[sequence]), cache.codes.shape[4]
    pages = cache.block_table[sequence, :-(-n // p)].long()
    values = cache.codes[layer, pages].double() * \
        torch.exp2(cache.exponents[layer, pages].double())[..., None, None]
    return values.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]


def _check_attend(cache, layer, q, sequences, counts, got, scale=D ** -0.5):
    group = q.shape[1] // cache.kv_heads
    start = 0
    for sequence, c in zip(sequences, counts):
        k, v = _values(cache, layer, sequence)
        for h in range(q.shape[1] if c else 0):
            want, _, bound = _rows(q[start:start + c, h].double(), k[h // group], v[h // group],
                                   k.shape[1] - c, scale)
            error = (got[start:start + c, h].double() - want).abs()
            assert bool((error <= bound).all()), (sequence, h, float((error / bound).max()))
        start += c


@pytest.mark.parametrize("page_tokens", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,counts", [
    (4, 2, [1, 1, 1, 1, 1, 1, 1]), (16, 1, [1, 2, 8, 1, 3, 0, 5]), (3, 3, [1, 1, 0, 1, 1, 1, 2]),
    (5, 1, [1, 7, 4, 1, 4, 0, 13]), (12, 4, [1, 15, 16, 63, 64, 65, 199])])
def test_attend_against_64_bits(attention, page_tokens, heads, kv_heads, counts):
    lengths = [1, 15, 16, 63, 64, 65, 199]
    cache = _filled(attention, lengths + [40], kv_heads, page_tokens, seed=heads)
    sequences = [3, 1, 6, 0, 5, 2, 4]
    counts = [min(c, lengths[s]) for c, s in zip(counts, sequences)]
    q = _normal(9, sum(counts), heads, D).to(torch.bfloat16)
    got = cache.attend(1, q, _int(sequences), _offsets(counts))
    assert cache.sync_status() == 0
    _check_attend(cache, 1, q, sequences, counts, got)
    assert torch.equal(cache.attend(1, q, _int(sequences), _offsets(counts)), got)


@pytest.mark.parametrize("lengths,counts,heads,kv_heads", [
    ([20000], [1], 16, 2), ([5000], [4], 8, 8), ([3000, 9, 1, 12345, 700], [1, 8, 1, 6, 2], 32, 2),
    ([700] * 70, [1] * 70, 8, 1), ([2500], [300], 16, 2), ([4000, 130], [8, 130], 32, 1)])
def test_attend_splits_long_sequences(attention, lengths, counts, heads, kv_heads):
    cache = _filled(attention, lengths, kv_heads, 64, seed=1, layers=1)
    q = (2 * _normal(10, sum(counts), heads, D)).to(torch.bfloat16)
    sequences = list(range(len(lengths)))
    got = cache.attend(0, q, _int(sequences), _offsets(counts), scale=0.05)
    assert cache.sync_status() == 0
    _check_attend(cache, 0, q, sequences, counts, got, scale=0.05)
    assert torch.equal(cache.attend(0, q, _int(sequences), _offsets(counts), scale=0.05), got)


def test_attend_pages_of_very_different_scales(attention):
    cache = _filled(attention, [500], 1, 64, seed=3, layers=1)
    pages = cache.block_table[0, :8].long()
    # values 2^64 apart; the largest keys stand where the values are small
    cache.exponents[0, pages, 1, 0] = torch.tensor([-32, 32, -32, 0, 32, -32, 5, -32], device="cuda").to(torch.int8)
    cache.exponents[0, pages, 0, 0] = torch.tensor([-3, -32, -5, -9, -32, -7, -6, -4], device="cuda").to(torch.int8)
    q = _normal(11, 3, 4, D).to(torch.bfloat16)
    got = cache.attend(0, q, _int([0]), _offsets([3]))
    _check_attend(cache, 0, q, [0], [3], got)


def test_attend_queries_of_any_size(attention):
    # rows whose elements lie many powers of two apart, rows of zeros, rows near bf16's ends
    cache = _filled(attention, [300, 300], 2, 32, seed=4, layers=1)
    q = _normal(12, 4, 8, D)
    q[0] *= torch.exp2(torch.linspace(-30, 0, D, device="cuda"))
    q[1] = 0
    q[2] *= 2.0 ** -100
    q[3] *= 2.0 ** 20
    q = q.to(torch.bfloat16)
    for row, scale in ((0, 0.1), (1, 0.1), (2, 0.1), (2, 2.0 ** 97), (3, 2.0 ** -23)):
        got = cache.attend(0, q[row:row + 1], _int([0]), _offsets([1]), scale=scale)
        _check_attend(cache, 0, q[row:row + 1], [0], [1], got, scale=scale)


def test_attend_keeps_what_is_masked_out(attention):
    heads, rows = 8, 6
    cache = _filled(attention, [133, 70], 2, 64, seed=5, layers=1)
    q = _normal(13, rows + 2, heads, D).to(torch.bfloat16)
    batch = (_int([0, 1]), _offsets([rows, 2]))
    clean = cache.attend(0, q, *batch)
    page = int(cache.block_table[0, 130 // 64])
    bits = cache.codes.view(torch.uint8)
    # a value that is no number at position 130: row 3 (position 130) and later ones see it
    before = int(bits[0, page, 1, 1, 130 % 64, 9])
    bits[0, page, 1, 1, 130 % 64, 9] = 0xFF
    got = cache.attend(0, q, *batch)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[3:rows, 4:, 9] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool(got[hit].float().isnan().all())
    bits[0, page, 1, 1, 130 % 64, 9] = before
    bits[0, page, 0, 0, 130 % 64, 9] = 0x7F  # and a key
    got = cache.attend(0, q, *batch)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[3:rows, :4] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool(got[hit].float().isnan().all())


def _code(x):
    """The nearest E4M3 value, ties to the even one."""
    _, power = torch.frexp(x)
    step = torch.exp2((power - 4).clamp(min=-9).double())
    return (torch.round(x / step) * step).clamp(-448, 448)


def _append_model(cache, layer, k, v, sequences, counts):
    codes, exponents = cache.codes.double(), cache.exponents.clone()
    p, start = cache.codes.shape[4], 0
    for sequence, c in zip(sequences, counts):
        n = int(cache.lengths[sequence])
        for place in range((n - c) // p, -(-n // p) if c else 0):
            page = int(cache.block_table[sequence, place])
            first, last = max(n - c, place * p), min(n, place * p + p)
            rows = slice(start + first - n + c, start + last - n + c)
            held = first - place * p
            for half, new in ((0, k), (1, v)):
                x = new[rows].double()
                finite = torch.where(x.isfinite(), x.abs(), 0.0).amax(dim=(0, 2))
                for h in range(x.shape[1]):
                    e = -32
                    while e < 32 and float(finite[h]) > 448 * 2.0 ** e:
                        e += 1
                    at = (layer, page, half, h)
                    if held:
                        e = max(e, int(exponents[at]))
                        codes[at][:held] = _code(codes[at][:held] * 2.0 ** (int(exponents[at]) - e))
                    fresh = _code(x[:, h] * 2.0 ** -e)
                    codes[at][held:last - place * p] = torch.where(x[:, h].isfinite(), fresh, math.nan)
                    exponents[at] = e
        start += c
    return codes, exponents


@pytest.mark.parametrize("page_tokens", [16, 32, 64, 128])
@pytest.mark.parametrize("lengths,counts", [
    ([1], [1]), ([130], [130]), ([64, 65, 0, 17], [1, 2, 0, 17]), ([700, 128, 129, 40], [3, 128, 100, 40])])
def test_append_is_exact(attention, page_tokens, lengths, counts):
    kv_heads = 3
    cache = _filled(attention, lengths, kv_heads, page_tokens, seed=7)
    rows = sum(counts)
    kv = _normal(15, rows, 2, kv_heads, D) * torch.exp2(8 * _normal(16, rows, 2, kv_heads, 1))
    kv[0, 0, 0, 0], kv[rows - 1, 1, 1, 1], kv[rows // 2, 0, 2, 2] = math.inf, math.nan, -math.inf
    kv[:, 1, 2] = 0
    kv = kv.to(torch.bfloat16)
    k, v = kv[:, 0], kv[:, 1]
    order = list(range(len(lengths)))[::-1]
    batch = (_int(order), _offsets([counts[i] for i in order]))
    codes, exponents = _append_model(cache, 1, k, v, order, [counts[i] for i in order])
    cache.append(1, k, v, *batch)
    assert cache.sync_status() == 0
    assert torch.equal(cache.exponents, exponents)
    got = cache.codes.double()
    assert bool(((got == codes) | (got.isnan() & codes.isnan())).all())


def test_append_at_the_ends_of_the_exponents(attention):
    cache = _filled(attention, [2, 2, 2], 1, 16, seed=8, layers=1)
    x = torch.zeros((6, 1, D), device="cuda")
    x[0, 0, :3] = torch.tensor([3e38, 1.0, -3e38])  # beyond 448 * 2^32: saturates
    x[2, 0, :3] = torch.tensor([1e-30, -1e-38, 0.0])  # below half of 2^-41: zero
    x[4, 0, :2] = torch.tensor([448.0 * 16, -450.0 * 16])  # on either side of a power
    x = x.to(torch.bfloat16)
    batch = (_int([0, 1, 2]), _offsets([2, 2, 2]))
    codes, exponents = _append_model(cache, 0, x, -x, [0, 1, 2], [2, 2, 2])
    cache.append(0, x, -x, *batch)
    assert torch.equal(cache.exponents, exponents)
    got = cache.codes.double()
    assert bool(((got == codes) | (got.isnan() & codes.isnan())).all())


def test_rows_appended_one_by_one_are_attended(attention):
    """A decode loop: every new row is written, then attends over itself and all before it."""
    kv_heads, heads, n = 2, 8, 70
    cache = attention.KvCache.allocate(1, 8, kv_heads, 3, 5, 16)
    kv = _normal(17, n, 2, kv_heads, D).to(torch.bfloat16)
    q = _normal(18, n, heads, D).to(torch.bfloat16)
    batch = (_int([2]), _offsets([1]))
    for t in range(n):
        cache.extend(*batch, rows=1)
        cache.append(0, kv[t:t + 1, 0], kv[t:t + 1, 1], *batch)
        got = cache.attend(0, q[t:t + 1], *batch)
        if t in (0, 1, 15, 16, 17, 40, 69):
            assert cache.sync_status() == 0 and int(cache.lengths[2]) == t + 1
            _check_attend(cache, 0, q[t:t + 1], [2], [1], got)
    # codes hold the rows to within their rounding: half a step of 1/8, and what a risen exponent lost
    stored = _values(cache, 0, 2).permute(2, 0, 1, 3)
    error = (stored - kv.double()).abs()
    assert float((error / (kv.double().abs() + 0.1)).max()) <= 2 ** -4 + 2 ** -8


# ---------------------------------------------------------------------------
# Pages
# ---------------------------------------------------------------------------

class Books:
    """The page operators on Python lists."""

    def __init__(self, cache):
        self.p = cache.codes.shape[4]
        self.table = [[] for _ in range(cache.block_table.shape[0])]
        self.lengths = [0] * len(self.table)
        self.references = [0] * cache.codes.shape[1]
        self.contents = [None] * len(self.references)  # a tag for what a page holds

    def _lowest(self, count):
        return [i for i, r in enumerate(self.references) if r == 0][:count]

    def extend(self, sequences, counts):
        for s, c in zip(sequences, counts):
            for page in self._lowest(-(-(self.lengths[s] + c) // self.p) - len(self.table[s])):
                self.references[page] = 1
                self.table[s].append(page)
            self.lengths[s] += c

    def free(self, sequences):
        for s in sequences:
            for page in self.table[s]:
                self.references[page] -= 1
            self.table[s], self.lengths[s] = [], 0

    def fork(self, parents, children):
        self.free(children)
        copies = iter(self._lowest(sum(self.lengths[s] % self.p != 0 for s in parents)))
        for parent, child in zip(parents, children):
            row = list(self.table[parent])
            if self.lengths[parent] % self.p:
                row[-1] = next(copies)
                self.contents[row[-1]] = self.contents[self.table[parent][-1]]
            for page in row:
                self.references[page] += 1
            self.table[child], self.lengths[child] = row, self.lengths[parent]

    def compact(self):
        live = sum(r > 0 for r in self.references)
        sources = [i for i, r in enumerate(self.references) if r and i >= live]
        targets = [i for i, r in enumerate(self.references) if not r and i < live]
        to = dict(zip(sources, targets))
        for source, target in to.items():
            self.references[target], self.references[source] = self.references[source], 0
            self.contents[target] = self.contents[source]
        self.table = [[to.get(page, page) for page in row] for row in self.table]

    def check(self, cache):
        assert cache.lengths.tolist() == self.lengths
        assert cache.references.tolist() == self.references
        width = cache.block_table.shape[1]
        assert cache.block_table.tolist() == [row + [0] * (width - len(row)) for row in self.table]
        tags = cache.codes.view(torch.uint8)[:, :, 1, -1, -1, -1].tolist()
        more = cache.exponents[:, :, 0, 0].tolist()
        for page, tag in enumerate(self.contents):
            if self.references[page] and tag is not None:
                for layer in range(cache.codes.shape[0]):
                    assert tags[layer][page] == (tag + layer) % 256
                    assert more[layer][page] == (tag + layer) % 64


def _tag(cache, books):
    """Gives every page contents of its own in every layer."""
    layers, pages = cache.codes.shape[:2]
    tags = torch.arange(pages, device="cuda")[None] + torch.arange(layers, device="cuda")[:, None]
    cache.codes.view(torch.uint8).copy_((tags % 256).to(torch.uint8)[:, :, None, None, None, None])
    cache.exponents.copy_((tags % 64).to(torch.int8)[:, :, None, None])
    books.contents = list(range(pages))


@pytest.mark.parametrize("pages,sequences,page_tokens,seed", [(40, 9, 16, 0), (200, 30, 32, 1),
                                                             (2500, 120, 64, 2)])
def test_books_of_pages(attention, pages, sequences, page_tokens, seed):
    import random
    rng = random.Random(seed)
    cache = attention.KvCache.allocate(3, pages, 2, sequences, 20, page_tokens)
    books = Books(cache)
    _tag(cache, books)
    for step in range(60):
        kind = rng.choice(["extend", "extend", "extend", "fork", "free", "compact"])
        some = rng.sample(range(sequences), rng.randint(1, sequences // 2))
        if kind == "extend":
            counts = [min(rng.choice([0, 1, 1, page_tokens, rng.randint(0, 5 * page_tokens)]),
                          20 * page_tokens - books.lengths[s]) for s in some]
            need = sum(-(-(books.lengths[s] + c) // page_tokens) - len(books.table[s])
                       for s, c in zip(some, counts))
            cache.extend(_int(some), _offsets(counts), rows=sum(counts))
            if need > books.references.count(0):
                assert cache.sync_status() == 6  # NMOE_ERR_CAPACITY, and nothing has changed
            else:
                books.extend(some, counts)
        elif kind == "fork" and len(some) > 1:
            children = some[:len(some) // 2 + 1]
            others = [s for s in range(sequences) if s not in children]
            parents = [rng.choice(others) for _ in children]
            own = sum(1 for page, r in enumerate(books.references)
                      if r and r == sum(row.count(page) for row in (books.table[s] for s in children)))
            need = sum(books.lengths[s] % page_tokens != 0 for s in parents)
            cache.fork(_int(parents), _int(children))
            if need > books.references.count(0) + own:
                assert cache.sync_status() == 6
            else:
                books.fork(parents, children)
        elif kind == "free":
            cache.free(_int(some))
            books.free(some)
        elif kind == "compact":
            cache.compact()
            books.compact()
        books.check(cache)
    assert cache.sync_status() == 0


def test_more_sequences_than_a_block_has_threads(attention):
    n, p = 2600, 16
    cache = attention.KvCache.allocate(1, 6000, 1, 2 * n, 3, p)
    books = Books(cache)
    _tag(cache, books)
    counts = [(7 * i) % 40 for i in range(n)]
    cache.extend(_int(list(range(n))), _offsets(counts), rows=sum(counts))
    books.extend(range(n), counts)
    books.check(cache)
    some = list(range(0, n, 3))
    cache.free(_int(some))
    books.free(some)
    cache.compact()
    books.compact()
    books.check(cache)
    parents = [i for i in range(n) if i % 3][:1500]
    children = list(range(n, n + len(parents)))
    cache.fork(_int(parents), _int(children))
    books.fork(parents, children)
    books.check(cache)
    assert cache.sync_status() == 0


def test_copy_pages(attention):
    cache = attention.KvCache.allocate(3, 50, 2, 2, 4, 32)
    books = Books(cache)
    _tag(cache, books)
    before = cache.codes.view(torch.uint8).clone(), cache.exponents.clone()
    sources, targets = list(range(0, 40, 2)), list(range(1, 41, 2))
    cache.copy_pages(_int(sources), _int(targets))
    assert cache.sync_status() == 0
    for got, was in zip((cache.codes.view(torch.uint8), cache.exponents), before):
        was[:, targets] = was[:, sources]
        assert torch.equal(got, was)


def test_a_forked_sequence_continues_on_its_own(attention):
    heads, kv_heads, p = 4, 2, 16
    cache = attention.KvCache.allocate(2, 20, kv_heads, 4, 6, p)
    n = 37
    kv = _normal(19, n + 2, 2, kv_heads, D).to(torch.bfloat16)
    prompt = (_int([0]), _offsets([n]))
    cache.extend(*prompt, rows=n)
    for layer in range(2):
        cache.append(layer, kv[:n, 0], kv[:n, 1], *prompt)
    cache.fork(_int([0, 0]), _int([2, 3]))
    both = (_int([3, 2]), _offsets([1, 1]))
    cache.extend(*both, rows=2)
    for layer in range(2):
        cache.append(layer, kv[n:, 0], kv[n:, 1], *both)
    assert cache.sync_status() == 0
    assert cache.references.tolist()[:6] == [3, 3, 1, 1, 1, 0]
    for layer in range(2):
        a, b, c = (_values(cache, layer, s) for s in (0, 2, 3))
        assert torch.equal(a[:, :, :32], b[:, :, :32]) and torch.equal(a[:, :, :32], c[:, :, :32])
        assert not torch.equal(b[:, :, -1], c[:, :, -1])
        q = _normal(20, 2, heads, D).to(torch.bfloat16)
        _check_attend(cache, layer, q, [3, 2], [1, 1], cache.attend(layer, q, *both))


def test_wrong_lists_change_nothing(attention):
    cache = _filled(attention, [100, 50, 30], 2, 32, seed=9)
    before = [t.clone() for t in (cache.block_table, cache.lengths, cache.references)]

    def unchanged():
        return all(torch.equal(a, b) for a, b in
                   zip(before, (cache.block_table, cache.lengths, cache.references)))

    for call in (lambda: cache.extend(_int([0, 3]), _offsets([1, 1]), rows=2),      # no such sequence
                 lambda: cache.extend(_int([1, 1]), _offsets([1, 1]), rows=2),      # named twice
                 lambda: cache.extend(_int([1]), _int([3, 1]), rows=3),             # offsets that fall
                 lambda: cache.free(_int([-1])), lambda: cache.free(_int([2, 2])),
                 lambda: cache.fork(_int([0]), _int([0])),                          # its own child
                 lambda: cache.fork(_int([0, 1]), _int([1, 2])),                    # a parent and a child
                 lambda: cache.fork(_int([7]), _int([1]))):
        call()
        assert cache.sync_status() == 1 and unchanged()
    cache.extend(_int([0]), _offsets([32 * 7]), rows=32 * 7)  # more than the pool and the table have
    codes = cache.codes.view(torch.uint8).clone()
    kv = torch.ones((1, 2, D), dtype=torch.bfloat16, device="cuda")
    cache.append(0, kv, kv, _int([0]), _offsets([1]))  # its row has no place: not written
    cache.free(_int([1]))
    assert cache.sync_status() == 6 and unchanged()
    assert torch.equal(cache.codes.view(torch.uint8), codes)
    # more new rows than the sequence has tokens, a page out of range: reported, nothing read there
    q = torch.ones((60, 4, D), dtype=torch.bfloat16, device="cuda")
    cache.attend(0, q, _int([1]), _offsets([60]))
    assert cache.sync_status() == 1
    cache.block_table[1, 0] = 10 ** 6
    cache.attend(0, q[:1], _int([1]), _offsets([1]))
    assert cache.sync_status() == 1
    cache.append(0, kv.repeat(50, 1, 1), kv.repeat(50, 1, 1), _int([1]), _offsets([50]))
    assert cache.sync_status() == 1
    cache.copy_pages(_int([0]), _int([10 ** 6]))
    assert cache.sync_status() == 1


def test_cache_refusals(attention, package):
    cache = attention.KvCache.allocate(2, 10, 2, 3, 4, 16)
    one, offsets = _int([0]), _offsets([1])
    q = torch.zeros((1, 4, D), dtype=torch.bfloat16, device="cuda")
    kv = q[:, :2]
    for call in (lambda: cache.attend(2, q, one, offsets), lambda: cache.attend(-1, q, one, offsets),
                 lambda: cache.attend(0, q[:, :3], one, offsets),
                 lambda: cache.attend(0, q, one, offsets, scale=math.inf),
                 lambda: cache.append(5, kv, kv, one, offsets),
                 lambda: cache.append(0, q, q, one, offsets)):
        with pytest.raises(package.NmoeError):
            call()
    for call in (lambda: cache.attend(0, q, one, one), lambda: cache.attend(0, q.float(), one, offsets),
                 lambda: cache.extend(one.long(), offsets, rows=1), lambda: cache.fork(one, offsets),
                 lambda: cache.copy_pages(one, offsets), lambda: cache.free(one.cpu()),
                 lambda: attention.KvCache.allocate(1, 4, 1, 1, 1, page_tokens=24),
                 lambda: attention.KvCache(cache.codes, cache.exponents[:1], cache.block_table,
                                           cache.lengths, cache.references)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(package.NmoeError):
        attention.KvCache.allocate(0, 4, 1, 1, 1)
    assert cache.attend(0, q[:0], _int([]), _offsets([])).shape == (0, 4, D)
    cache.extend(_int([]), _offsets([]), rows=0)
    cache.free(_int([]))
    assert cache.sync_status() == 0


def test_a_decode_step_is_replayed_from_a_graph(attention):
    kv_heads, heads, p = 2, 8, 16
    cache = attention.KvCache.allocate(1, 64, kv_heads, 2, 20, p)
    batch = (_int([0, 1]), _offsets([1, 1]))
    k, v = (torch.zeros((2, kv_heads, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros((2, heads, D), dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)

    def step():
        cache.extend(*batch, rows=2)
        cache.append(0, k, v, *batch)
        cache.attend(0, q, *batch, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(40):
        for t, seed in ((k, 3), (v, 4), (q, 5)):
            t.copy_(_normal(100 * i + seed, *t.shape).to(torch.bfloat16))
        graph.replay()
    assert cache.sync_status() == 0 and cache.lengths.tolist() == [41, 41]
    _check_attend(cache, 0, q, [0, 1], [1, 1], out)


@pytest.mark.parametrize("heads", [4, 32, 64])
def test_two_caches_on_two_streams(attention, heads):
    """Both calls' sequences are cut between blocks that the other call may keep from running."""
    caches, queries, alone = [], [], []
    for seed in range(2):
        cache = attention.KvCache.allocate(1, 64, 2, 3, 40, page_tokens=64)
        lengths = [1500, 7, 900]
        kv = _normal(40 + seed, 2, sum(lengths), 2, D).to(torch.bfloat16)
        everyone = _int([0, 1, 2])
        cache.extend(everyone, _offsets(lengths), sum(lengths))
        cache.append(0, kv[0], kv[1], everyone, _offsets(lengths))
        caches.append(cache)
        queries.append(_normal(50 + seed, 3, heads, D).to(torch.bfloat16))
        alone.append(cache.attend(0, queries[seed], everyone, _offsets([1, 1, 1])))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    offsets, results = _offsets([1, 1, 1]), [[], []]
    for _ in range(50):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(caches[i].attend(0, queries[i], everyone, offsets))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r, alone[i]) for r in results[i])
        assert caches[i].sync_status() == 0


def test_a_cache_of_more_than_4_gb(attention):
    """The last pages of a large pool, of which something else holds the others, do what those of a
    small pool do."""
    kv_heads, heads, few, pages, layers = 2, 8, 24, 75000, 2
    lengths = [130, 0, 300]
    kv = _normal(60, sum(lengths), 2, kv_heads, D).to(torch.bfloat16)
    more = _normal(61, 4, 2, kv_heads, D).to(torch.bfloat16)
    q = _normal(62, 4, heads, D).to(torch.bfloat16)
    caches, results = [], []
    for n in (few, pages):
        cache = attention.KvCache.allocate(layers, n, kv_heads, 4, 8, 64)
        cache.references[:n - few] = 1
        prompts = (_int([0, 1, 2]), _offsets(lengths))
        cache.extend(*prompts, rows=sum(lengths))
        for layer in range(layers):
            cache.append(layer, kv[:, 0], kv[:, 1], *prompts)
        cache.fork(_int([2]), _int([3]))
        step = (_int([3, 0, 2]), _offsets([2, 1, 1]))
        cache.extend(*step, rows=4)
        for layer in range(layers):
            cache.append(layer, more[:, 0], more[:, 1], *step)
            results.append(cache.attend(layer, q, *step))
        cache.free(_int([0]))
        cache.compact()
        results.append(cache.attend(layers - 1, q[:3], _int([3, 2]), _offsets([2, 1])))
        assert cache.sync_status() == 0
        caches.append(cache)
    small, large = caches
    assert large.codes.numel() > 2 ** 32
    assert torch.equal(large.block_table[2:] - small.block_table[2:],
                       (small.block_table[2:] > 0) * (pages - few) +
                       (small.block_table[2:] == 0) * large.block_table[2:])
    assert torch.equal(large.references[-few:], small.references)
    assert torch.equal(large.exponents[:, -few:], small.exponents)
    assert torch.equal(large.codes[:, -few:].view(torch.uint8), small.codes.view(torch.uint8))
    for a, b in zip(results[:3], results[3:]):
        assert torch.equal(a, b)
    del small
    _check_attend(large, 1, torch.cat((q[:2], q[3:])), [3, 2], [2, 1],
                  large.attend(1, torch.cat((q[:2], q[3:])), _int([3, 2]), _offsets([2, 1])))


def test_prefill_of_rows_beyond_4_gb(attention):
    """Prompts at the end of a batch whose queries and results are larger than 4 GB."""
    rows, heads, kv_heads, lengths = 600000, 32, 2, [200, 0, 77]
    used = sum(lengths)
    small = [_normal(70 + i, used, h, D).to(torch.bfloat16) for i, h in enumerate((heads, kv_heads, kv_heads))]
    large = [torch.zeros((rows,) + t.shape[1:], dtype=t.dtype, device="cuda") for t in small]
    for a, b in zip(large, small):
        a[-used:] = b
    got, lse = attention.attention_prefill(*large, _offsets(lengths) + (rows - used), return_lse=True)
    want, sums = attention.attention_prefill(*small, _offsets(lengths), return_lse=True)
    assert attention.prefill_sync_status() == 0
    assert torch.equal(got[-used:], want) and torch.equal(lse[-used:], sums)
    _check_prefill(*small, lengths, got[-used:], lse[-used:])


@pytest.mark.parametrize("lengths,counts,heads,kv_heads", [
    ([30000], [8], 16, 1), ([9000, 20011], [3, 5], 8, 1), ([40000], [2], 18, 1), ([1000] * 40, [7] * 40, 32, 2)])
def test_attend_joins_many_pieces_of_many_rows(attention, lengths, counts, heads, kv_heads):
    cache = _filled(attention, lengths, kv_heads, 64, seed=2, layers=1)
    q = (2 * _normal(11, sum(counts), heads, D)).to(torch.bfloat16)
    batch = (_int(list(range(len(lengths)))), _offsets(counts))
    got = cache.attend(0, q, *batch, scale=0.05)
    assert cache.sync_status() == 0
    _check_attend(cache, 0, q, list(range(len(lengths))), counts, got, scale=0.05)
    assert torch.equal(cache.attend(0, q, *batch, scale=0.05), got)
