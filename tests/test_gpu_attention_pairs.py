"""GPU tests of attention over shared tokens by the kernel for more than 128 rows of queries to a group and key head.

Tolerances are those of tests/test_gpu_attention_shared.py: its kernel's weights are within 2^-11 of themselves or 2^-25 of
the largest that its reference allows (2^8), which the bounds there hold with room."""
import importlib
import math
import random

import pytest
import torch

from test_gpu_attention import _int, _normal, _offsets, _values
from test_gpu_attention_shared import _attend, _check, _edges, _expected_shared, _shared_cache

pytestmark = pytest.mark.gpu

D = 128


@pytest.fixture(scope="module")
def attention(package):
    return importlib.import_module("nemotron_inference_b200.attention")


def _check_some(cache, q, counts, got, which):
    """Entries `which`, those of sequences of the same number."""
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    for i in which:
        rows = slice(starts[i], starts[i + 1])
        _check(cache, 0, q[rows], [i], counts[i:i + 1], got[rows])


@pytest.mark.parametrize("prompts", [[130], [128, 131, 300], [257, 129]])
@pytest.mark.parametrize("heads,members", [(144, 5), (272, 4)])
def test_many_units_of_a_tile_each(attention, prompts, heads, members):
    """Short prompts of many groups: a block has several (group, key head, rows) one after another, most of them of a
    single tile, the rows of one tile or of two."""
    kv_heads, n = 4, 150
    groups = [(prompts[i % len(prompts)], [1 + (i + j) % 3 for j in range(members)]) for i in range(n)]
    cache = _shared_cache(attention, groups, [], kv_heads, 64, seed=len(prompts))
    q = _normal(30, n * members, heads, D).to(torch.bfloat16)
    sequences, counts = list(range(n * members)), [1] * (n * members)
    assert members * heads // kv_heads > 128
    first, shared = _attend(cache, 0, q, sequences, counts, _edges(groups))
    assert cache.sync_status() == 0 and int(shared.min()) >= 128
    _check_some(cache, q, counts, first, random.Random(heads).sample(sequences, 12))
    for _ in range(5):
        assert torch.equal(_attend(cache, 0, q, sequences, counts, _edges(groups))[0], first)
    assert cache.sync_status() == 0


# (prompt, tokens of each member beside it), of more than 128 rows to a group at `_HEADS` query heads and one key head
_HEADS = 40
_GROUPS = [(300, [20, 30, 3, 9]), (260, [4, 4, 70])]
_COUNTS = [2, 1, 3, 1, 1, 2, 1]


def _problem(attention, seed, page_tokens=64, layers=1, scale_of_q=1.0):
    cache = _shared_cache(attention, _GROUPS, [], 1, page_tokens, seed=seed, layers=layers)
    q = (scale_of_q * _normal(seed + 1, sum(_COUNTS), _HEADS, D)).to(torch.bfloat16)
    assert -(-sum(_COUNTS) // len(_GROUPS)) * _HEADS > 128
    return cache, q, (_int(list(range(len(_COUNTS)))), _offsets(_COUNTS)), _edges(_GROUPS)


def test_no_numbers_reach_who_sees_them(attention):
    """A key or value of the shared tokens that is no number, in each of a tile's places and at each of their ends, reaches
    all rows of its group and no other; a query that is none, its row."""
    cache, q, batch, edges = _problem(attention, 6)
    sequences = list(range(len(_COUNTS)))
    clean, shared = _attend(cache, 0, q, sequences, _COUNTS, edges)
    assert shared.tolist() == [256] * 7
    _check(cache, 0, q, sequences, _COUNTS, clean)
    bits = cache.codes.view(torch.uint8)
    first_rows = sum(_COUNTS[:4])
    for code in (0x7F, 0xFF):
        for sequence, rows in ((1, slice(0, first_rows)), (5, slice(first_rows, None))):
            for position, dim in ((0, 0), (77, 11), (127, 127), (128, 64), (200, 5), (255, 90)):
                for half in (0, 1):
                    at = (0, int(cache.block_table[sequence, position // 64]), half, 0, position % 64, dim)
                    before = int(bits[at])
                    bits[at] = code
                    got = cache.attend_shared(0, q, *batch, edges, shared)
                    bits[at] = before
                    hit = torch.zeros_like(clean, dtype=torch.bool)
                    hit[rows, :, slice(None) if half == 0 else dim] = True
                    assert torch.equal(got[~hit], clean[~hit]) and bool(got[hit].float().isnan().all()), (position, half)
    for value in (float("nan"), float("inf"), -float("inf")):
        bad = q.clone()
        bad[3, 17, 40] = value
        got = cache.attend_shared(0, bad, *batch, edges, shared)
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[3, 17] = True
        assert torch.equal(got[~hit], clean[~hit]) and bool(got[hit].float().isnan().all())
    assert cache.sync_status() == 0


@pytest.mark.parametrize("page_tokens", [16, 64, 128])
@pytest.mark.parametrize("low,high", [(-12, 4), (-40, -30), (10, 20)])
def test_powers_of_pages_far_apart(attention, page_tokens, low, high):
    """Pages' powers differ within a tile and from tile to tile, those of keys and of values for themselves."""
    cache, q, batch, edges = _problem(attention, 7, page_tokens)
    g = torch.Generator().manual_seed(low + 100)
    keys = torch.randint(-12, 1, cache.exponents[:, :, 0].shape, generator=g) - 6
    values = torch.randint(low, high + 1, cache.exponents[:, :, 1].shape, generator=g)
    cache.exponents[:, :, 0], cache.exponents[:, :, 1] = keys.to(torch.int8).cuda(), values.to(torch.int8).cuda()
    got, shared = _attend(cache, 0, q, list(range(7)), _COUNTS, edges, scale=0.02)
    assert shared.tolist() == [256] * 7 and cache.sync_status() == 0
    start = 0
    for sequence, c in enumerate(_COUNTS):
        _check_far(cache, q[start:start + c], sequence, c, got[start:start + c], 0.02)
        start += c


def _check_far(cache, q, sequence, c, got, scale):
    """With powers apart: a weight is relative to the largest of weight times 2^power of its page's values, which is
    what a row's reference goes by; what is off by 2^-20.5 of that is multiplied with codes, of at most 448."""
    n, p = int(cache.lengths[sequence]), cache.codes.shape[4]
    values = _values(cache, 0, sequence)
    power = torch.exp2(cache.exponents[0, cache.block_table[sequence, :-(-n // p)].long(), 1, 0].double()).repeat_interleave(p)[:n]
    k, v = values[0][0], values[1][0]
    seen = torch.arange(n, device="cuda")[None] <= n - c + torch.arange(c, device="cuda")[:, None]
    for h in range(q.shape[1]):
        rows = q[:, h].double()
        scores = ((rows @ k.T) * scale).masked_fill(~seen, -math.inf)
        w = torch.softmax(scores, dim=1)
        delta = scale * 2.0 ** -17 * rows.abs().amax(1, keepdim=True) * k.abs().sum(1).max()
        largest = (w * power).amax(1, keepdim=True)
        bound = (2.5 * 2 ** -8 + 2.2 * delta) * (w @ v.abs()) + 2 ** -20.5 * largest * (v.abs() / power[:, None]).sum(0)
        error = (got[:, h].double() - w @ v).abs()
        assert bool((error <= bound).all()), (sequence, h, float((error / bound).max()))


@pytest.mark.parametrize("later", [128, 200, 255])
def test_scores_that_rise_far(attention, later):
    """Rows whose scores in a later tile of the shared tokens lie thousands of orders above those before, others whose do
    not, and rows of which all shared tokens lie far below or above their own."""
    cache, q, batch, edges = _problem(attention, 8)
    page, place = later // 64, later % 64
    codes = cache.codes[0, int(cache.block_table[0, page]), 0, 0]
    for exponent, scale in ((-6, 30.0), (0, 30.0), (0, 500.0), (-6, 0.05)):
        cache.exponents[0, int(cache.block_table[0, page]), 0] = exponent
        for sign in (1.0, -1.0):
            kept = codes[place].clone()
            codes[place] = (sign * 448 * torch.sign(q[0, 0].float())).to(torch.float8_e4m3fn)
            got, shared = _attend(cache, 0, q, list(range(7)), _COUNTS, edges, scale=scale)
            codes[place] = kept
            assert shared.tolist() == [256] * 7 and cache.sync_status() == 0
            assert bool(got.isfinite().all())
            if sign > 0 and scale >= 30.0:
                # row 0, head 0: nothing but that token's value
                v = cache.codes[0, int(cache.block_table[0, page]), 1, 0, place].double() * \
                    2.0 ** float(cache.exponents[0, int(cache.block_table[0, page]), 1, 0])
                assert bool(((got[0, 0].double() - v).abs() <= 2.5 * 2.0 ** -8 * v.abs()).all())
            if scale < 1.0:
                codes[place] = (sign * 448 * torch.sign(q[0, 0].float())).to(torch.float8_e4m3fn)
                _check(cache, 0, q, list(range(7)), _COUNTS, got, scale=scale)
                codes[place] = kept


def test_recorded_and_replayed_while_lengths_change(attention):
    cache, q, batch, edges = _problem(attention, 9)
    out, shared = torch.empty_like(q), torch.empty(7, dtype=torch.int32, device="cuda")

    def step():
        cache.find_shared(*batch, edges, out=shared)
        cache.attend_shared(0, q, *batch, edges, shared, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    cache.lengths.sub_(torch.tensor([5, 20, 0, 0, 1, 2, 69], dtype=torch.int32, device="cuda"))
    q.copy_(_normal(40, *q.shape))
    graph.replay()
    replayed = out.clone()
    assert shared.tolist() == [256] * 7
    _check(cache, 0, q, list(range(7)), _COUNTS, replayed)
    cache.lengths[6] = 200  # beyond its group's page 3: shared by fewer tokens
    graph.replay()
    assert shared.tolist() == [256] * 4 + [128] * 3
    _check(cache, 0, q, list(range(7)), _COUNTS, out)
    replayed = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, replayed) and cache.sync_status() == 0


def test_wrong_plans_leave_zeros_and_a_status(attention):
    cache, q, batch, edges = _problem(attention, 10)
    right = cache.find_shared(*batch, edges)
    clean = cache.attend_shared(0, q, *batch, edges, right)
    own = sum(_COUNTS[:4])  # rows of the first group
    for entry, value in ((0, 640), (1, 100), (1, -128), (1, 128), (0, 2 ** 30)):
        shared = right.clone()
        shared[entry] = value
        got = cache.attend_shared(0, q, *batch, edges, shared)
        assert cache.sync_status() == 1
        assert torch.equal(got[own:], clean[own:])
        assert bool((got[slice(0, 2) if entry == 0 else slice(2, 3)] == 0).all())
    for bad in ([0, 4, 99], [-1, 4, 7], [0, 6, 4]):
        cache.attend_shared(0, q, *batch, _int(bad), right)
        assert cache.sync_status() == 1
    got = cache.attend_shared(0, q, _int([0, 99, 2, 3, 4, 5, 6]), batch[1], edges, right)
    assert cache.sync_status() == 1 and bool((got[2:3] == 0).all()) and torch.equal(got[own:], clean[own:])
    cache.extend(_int([99]), _offsets([1]), 1)  # books that have failed
    assert bool((cache.attend_shared(0, q, *batch, edges, right) == 0).all())
    assert cache.sync_status() == 1
    assert torch.equal(cache.attend_shared(0, q, *batch, edges, right), clean) and cache.sync_status() == 0


def test_batches_whose_entries_are_all_wrong_or_empty(attention):
    """Zeros and a status, there before what follows the call reads them; rows of no entry as they were."""
    cache, q, batch, edges = _problem(attention, 11)
    shared = cache.find_shared(*batch, edges)
    for _ in range(20):
        out = torch.full_like(q, 3.0)
        cache.attend_shared(0, q, _int([99] * 7), batch[1], edges, shared, out=out)
        read = out.clone()
        assert bool((read == 0).all())
        out.fill_(3.0)
        cache.attend_shared(0, q, batch[0], _int([0] * 8), edges, shared, out=out)
        assert bool((out == 3.0).all())
    assert cache.sync_status() == 1


def test_two_calls_on_two_streams(attention):
    """Two caches, a stream each, at the same time; one takes the kernel for fewer rows."""
    problems = [_problem(attention, 12), _problem(attention, 13)]
    shared = [c.find_shared(*batch, edges) for c, _, batch, edges in problems]
    queries = [problems[0][1], problems[1][1][:, :8].contiguous()]
    call = lambda i: problems[i][0].attend_shared(0, queries[i], *problems[i][2], problems[i][3], shared[i])  # noqa: E731
    alone = [call(0), call(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append(call(i))
        torch.cuda.synchronize()
        assert torch.equal(got[0], alone[0]) and torch.equal(got[1], alone[1])
    assert all(c.sync_status() == 0 for c, _, _, _ in problems)


def test_two_graphs_of_one_cache(attention):
    """Two layers, a recording each, replayed one after the other in both orders."""
    cache, q, batch, edges = _problem(attention, 14, layers=2)
    shared = cache.find_shared(*batch, edges)
    want = [cache.attend_shared(layer, q, *batch, edges, shared) for layer in (0, 1)]
    outs, graphs = [torch.empty_like(q) for _ in want], []
    torch.cuda.synchronize()
    for layer in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.attend_shared(layer, q, *batch, edges, shared, out=outs[layer])
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for out in outs:
            out.zero_()
        for i in order:
            graphs[i].replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert cache.sync_status() == 0


def test_sequences_in_any_order_wide_rows_and_rows_of_no_entry(attention):
    """Queries that lie among other columns, entries without rows, entries of no group before and behind, two key heads."""
    groups = [(600, [30, 40, 50, 60]), (300, [10, 20, 5]), (129, [2, 2])]
    cache = _shared_cache(attention, groups, [77, 900], 2, 32, seed=15, layers=2)
    sequences = [10, 2, 0, 3, 1, 6, 4, 5, 7, 8, 9]
    counts = [3, 4, 0, 5, 6, 4, 0, 3, 1, 1, 3]
    edges = _int([1, 5, 8, 10])
    heads, rows = 2 * 36, sum(counts)
    wide = _normal(16, rows + 5, heads + 8, D).to(torch.bfloat16)
    q = wide[:, 4:heads + 4]
    assert -(-(rows + 5) // 3) * 36 > 128 and not q.is_contiguous()
    out = torch.full((rows + 5, heads, D), 5.0, dtype=torch.bfloat16, device="cuda")
    got, shared = _attend(cache, 1, q, sequences, counts, edges, out=out)
    assert got is out and bool((out[rows:] == 5.0).all()) and cache.sync_status() == 0
    assert shared.tolist() == _expected_shared(cache, sequences, counts, edges.tolist())
    assert shared.tolist()[0] == 0 and shared.tolist()[1] == 512 and shared.tolist()[5] == 256
    _check(cache, 1, q, sequences, counts, got)
