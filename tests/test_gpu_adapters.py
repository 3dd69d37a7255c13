"""GPU tests of low-rank adapters against 64 bits.

Tolerances, per element: the result is bf16, half a step 2^-8 of it at most (just above a power of two).  What the
adapter adds is sum_j s t_j b_j with t_j within 2^-17 of itself (two bf16 terms) and FP32 sums t_j off by at most
inner 2^-24 sum |x a| (a step of the sum each): s sum_j (2^-17 |t_j| + inner 2^-24 (|x| |a|^T)_j) |b_j|, and as much again
for the sums over the ranks (2 rank 2^-24 sum |t b|, below 2^-16)."""
import importlib
import random

import pytest
import torch

from test_gpu_attention import _int, _normal, _offsets

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def adapters(package):
    return importlib.import_module("nemotron_inference_b200.adapters")


def _pool(adapters, n, rank, inner, outer, seed=1):
    a = (_normal(seed, n, rank, inner) * inner ** -0.5).to(torch.bfloat16)
    b = (_normal(seed + 1, n, outer, rank) * rank ** -0.5).to(torch.bfloat16)
    return adapters.AdapterPool(a, b, 0.5 + _normal(seed + 2, n).abs())


def _check(pool, x, y, ids, counts, got):
    start = 0
    for which, c in zip(ids, counts):
        rows = slice(start, start + c)
        start += c
        if which < 0:
            assert torch.equal(got[rows], y[rows])
            continue
        a, b, s = pool.a[which].double(), pool.b[which].double(), float(pool.scales[which])
        t = x[rows].double() @ a.T
        want = y[rows].double() + s * (t @ b.T)
        off = (2.0 ** -17 + 2.0 ** -16) * t.abs() + pool.inner * 2.0 ** -24 * (x[rows].double().abs() @ a.abs().T)
        bound = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * s * (off @ b.abs().T) + 1e-30
        error = (got[rows].double() - want).abs()
        assert bool((error <= bound).all()), (which, c, float((error / bound).max()))


def _inputs(pool, rows, seed=7):
    return _normal(seed, rows, pool.inner).to(torch.bfloat16), (2 * _normal(seed + 1, rows, pool.outer)).to(torch.bfloat16)


@pytest.mark.parametrize("counts", [[1], [3], [1] * 40, [16, 17, 1, 0, 15], [128], [129, 1, 0, 300], [5, 127, 128, 2],
                                    [1000]])
@pytest.mark.parametrize("rank,inner,outer", [(8, 64, 128), (16, 2688, 4608), (24, 200, 328), (32, 8, 8), (64, 4096, 2688),
                                              (72, 520, 136), (128, 1000, 1048)])
def test_against_64_bits(adapters, counts, rank, inner, outer):
    pool = _pool(adapters, 7, rank, inner, outer)
    rng = random.Random(sum(counts) + rank)
    ids = [rng.randrange(-1, 7) for _ in counts]
    ids[0] = 6  # the last one: behind its rows lies nothing
    x, y = _inputs(pool, sum(counts))
    before = y.clone()
    got = pool.add(x, y, _int(ids), _offsets(counts))
    assert pool.sync_status() == 0 and torch.equal(y, before)
    _check(pool, x, y, ids, counts, got)
    assert torch.equal(pool.add(x, y, _int(ids), _offsets(counts)), got)  # the same bits
    assert pool.add(x, y, _int(ids), _offsets(counts), out=y) is y and torch.equal(y, got)


def test_many_entries_and_rows(adapters):
    pool = _pool(adapters, 3, 16, 256, 384)
    for counts in ([1] * 700, [random.Random(3).randint(0, 5) for _ in range(1500)], [4000], [900] * 4):
        ids = [i % 4 - 1 for i in range(len(counts))]
        x, y = _inputs(pool, sum(counts))
        _check(pool, x, y, ids, counts, pool.add(x, y, _int(ids), _offsets(counts)))
    assert pool.sync_status() == 0


def test_rows_of_wider_tensors_and_rows_of_no_entry(adapters):
    pool = _pool(adapters, 4, 16, 320, 264)
    wide_x, wide_y = _normal(3, 90, 400).to(torch.bfloat16), _normal(4, 90, 600).to(torch.bfloat16)
    x, y = wide_x[:, 40:360], wide_y[:, 8:272]
    out = torch.full((90, 512), 3.0, dtype=torch.bfloat16, device="cuda")
    before = wide_y.clone()
    got = pool.add(x, y, _int([2, 0]), _int([5, 40, 80]), out=out[:, 16:280])
    assert got.data_ptr() == out[:, 16:280].data_ptr()
    _check(pool, x[5:80], y[5:80], [2, 0], [35, 40], got[5:80])
    assert bool((out[:5] == 3).all() and (out[80:] == 3).all() and (out[:, :16] == 3).all() and (out[:, 280:] == 3).all())
    pool.add(x, y, _int([2, 0]), _int([5, 40, 80]), out=y)  # in its place
    assert torch.equal(y[5:80], got[5:80])
    wide_y[:, 8:272][5:80] = before[:, 8:272][5:80]
    assert torch.equal(wide_y, before)
    assert pool.sync_status() == 0


def test_no_numbers_stay_in_their_rows(adapters):
    pool = _pool(adapters, 3, 16, 128, 256)
    x, y = _inputs(pool, 40)
    clean = pool.add(x, y, _int([0, 1, -1]), _int([0, 15, 30, 40]))
    x[7, 3], x[35, 0], y[20, 9] = float("nan"), float("nan"), float("inf")
    pool.b[2] = float("nan")  # an adapter that nobody has
    pool.a[2] = float("nan")
    got = pool.add(x, y, _int([0, 1, -1]), _int([0, 15, 30, 40]))
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[7] = True
    hit[20, 9] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool(got[7].float().isnan().all()) and float(got[20, 9]) == float("inf")
    pool.b[1, 100] = float("nan")  # a column of its rows
    got = pool.add(x, y, _int([0, 1, -1]), _int([0, 15, 30, 40]))
    hit[15:30, 100] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool(got[15:30, 100].float().isnan().all())


def test_wrong_lists_are_reported(adapters):
    pool = _pool(adapters, 3, 8, 64, 128)
    x, y = _inputs(pool, 30)
    clean = pool.add(x, y, _int([0, 1, 2]), _int([0, 10, 20, 30]))
    got = pool.add(x, y, _int([0, 3, 2]), _int([0, 10, 20, 30]))  # an id that is none: none
    assert pool.sync_status() == 1 and torch.equal(got[10:20], y[10:20]) and torch.equal(got[20:], clean[20:])
    got = pool.add(x, y, _int([0, -2, 2]), _int([0, 10, 20, 30]))
    assert pool.sync_status() == 1 and torch.equal(got[10:20], y[10:20])
    for offsets in ([0, 10, 31, 30], [0, 10, 5, 30], [-1, 10, 20, 30]):
        out = torch.full_like(y, 9.0)
        pool.add(x, y, _int([0, 1, 2]), _int(offsets), out=out)
        assert pool.sync_status() == 1
        for i, (from_, to) in enumerate(zip(offsets, offsets[1:])):
            if 0 <= from_ <= to <= 30 and offsets != [0, 10, 5, 30]:
                assert torch.equal(out[from_:to], clean[from_:to]) if i != 2 or from_ == 20 else True
    assert torch.equal(pool.add(x, y, _int([0, 1, 2]), _int([0, 10, 20, 30])), clean) and pool.sync_status() == 0


def test_recorded_and_on_another_stream(adapters):
    pool = _pool(adapters, 5, 16, 512, 640)
    x, y = _inputs(pool, 64)
    ids, offsets, out = _int([0, 1, 2]), _int([0, 20, 30, 64]), torch.empty_like(y)
    pool.add(x, y, ids, offsets, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.add(x, y, ids, offsets, out=out)
    x2, y2 = _inputs(pool, 64, seed=30)
    x.copy_(x2)
    y.copy_(y2)
    ids.copy_(_int([4, -1, 3]))
    offsets.copy_(_int([0, 1, 50, 64]))
    graph.replay()
    replayed = out.clone()
    _check(pool, x2, y2, [4, -1, 3], [1, 49, 14], replayed)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = pool.add(x, y, ids, offsets)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(aside, replayed) and pool.sync_status() == 0


def test_refusals(adapters, package):
    pool = _pool(adapters, 3, 8, 64, 128)
    x, y = _inputs(pool, 8)
    ids, offsets = _int([0]), _int([0, 8])
    for bad in (dict(x=x.float()), dict(x=x[:, :56]), dict(y=y[:4]), dict(y=y.cpu()), dict(ids=ids.long()),
                dict(offsets=_int([0])), dict(out=y.float()), dict(x=x[0]), dict(ids=ids[:0], offsets=_int([0])),
                dict(x=_normal(1, 8, 80).to(torch.bfloat16)[:, 4:68]), dict(y=y.t().contiguous().t())):
        arguments = dict(x=x, y=y, ids=ids, offsets=offsets)
        arguments.update(bad)
        with pytest.raises(ValueError):
            pool.add(**arguments)
    a, b = pool.a, pool.b
    for bad in (dict(a=a.float()), dict(a=a[:, :4].contiguous(), b=b[:, :, :4].contiguous()), dict(b=b[:2]), dict(a=a.cpu()),
                dict(scales=pool.scales[:2]), dict(a=a[0]), dict(b=b[:, :, ::2]),
                dict(a=torch.zeros((1, 136, 64), dtype=torch.bfloat16, device="cuda"),
                     b=torch.zeros((1, 128, 136), dtype=torch.bfloat16, device="cuda"))):
        arguments = dict(a=a, b=b, scales=pool.scales)
        arguments.update(bad)
        with pytest.raises(ValueError):
            adapters.AdapterPool(**arguments)
    assert pool.add(x[:0], y[:0], ids, _int([0, 0])).shape == (0, 128)
