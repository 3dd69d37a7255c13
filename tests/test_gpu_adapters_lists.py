"""GPU tests of low-rank adapters: lists that are wrong leave the rows that they should not touch as they were, and results
that may not lie where they are asked for.  Tolerances: those of tests/test_gpu_adapters.py."""
import importlib

import pytest
import torch

from test_gpu_adapters import _check, _inputs, _pool
from test_gpu_attention import _int

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def adapters(package):
    return importlib.import_module("nemotron_inference_b200.adapters")


@pytest.mark.parametrize("offsets", [[0, 10, 31, 30], [0, 10, 5, 30], [-1, 10, 20, 30], [10, 31, 30, 30], [0, 7, 7, 2 ** 31 - 1],
                                     [30, 20, 10, 0], [-2 ** 31, 4, 9, 12], [0, 12, 12, 10], [3, 40, 50, 60]])
def test_rows_of_entries_that_are_none_stay_as_they_were(adapters, offsets):
    pool = _pool(adapters, 3, 8, 64, 128)
    x, y = _inputs(pool, 30)
    ids = [0, 1, 2]
    valid = [i for i in range(3) if 0 <= offsets[i] <= offsets[i + 1] <= 30]
    covered = [sum(offsets[i] <= r < offsets[i + 1] for i in valid) for r in range(30)]
    out = torch.full_like(y, 9.0)
    pool.add(x, y, _int(ids), _int(offsets), out=out)
    assert pool.sync_status() == 1
    for r in range(30):
        if covered[r] == 0:
            assert bool((out[r] == 9.0).all()), r
        elif covered[r] == 1:  # (in two entries: either one's)
            i = next(i for i in valid if offsets[i] <= r < offsets[i + 1])
            _check(pool, x[r:r + 1], y[r:r + 1], [ids[i]], [1], out[r:r + 1])


def test_many_wrong_entries(adapters):
    """Among 300 entries of 7 rows some whose offsets lie beside the rows: their neighbours have the same edges."""
    pool = _pool(adapters, 3, 16, 128, 264)
    n = 300
    x, y = _inputs(pool, 7 * n)
    offsets = [7 * i for i in range(n + 1)]
    for i in (0, 40, 41, 155, 299):
        offsets[i] = -5 if i % 2 else 7 * n + 100
    ids = [i % 4 - 1 for i in range(n)]
    out = torch.full_like(y, 9.0)
    pool.add(x, y, _int(ids), _int(offsets), out=out)
    assert pool.sync_status() == 1
    for i in range(n):
        rows = slice(7 * i, 7 * i + 7)
        if 0 <= offsets[i] <= offsets[i + 1] <= 7 * n:
            _check(pool, x[rows], y[rows], ids[i:i + 1], [7], out[rows])
        else:
            assert bool((out[rows] == 9.0).all()), i


def test_results_over_other_rows_are_refused(adapters, package):
    """`out` may be y, which means y's rows: not what begins where y does and has its rows elsewhere."""
    pool = _pool(adapters, 2, 8, 128, 128)
    whole = torch.zeros((16, 256), dtype=torch.bfloat16, device="cuda")
    x, _ = _inputs(pool, 16)
    ids, offsets = _int([-1]), _int([0, 16])
    near = whole.view(-1)[:16 * 128].view(16, 128)
    for y, out in ((whole[:, :128], near), (near, whole[:, :128])):
        with pytest.raises(package.NmoeError) as info:
            pool.add(x, y, ids, offsets, out=out)
        assert info.value.status == 1
    assert pool.add(x, whole[:, :128], ids, offsets, out=whole[:, 128:]).data_ptr() == whole[:, 128:].data_ptr()
    assert pool.sync_status() == 0


def test_two_calls_on_two_streams(adapters):
    """One pool and a word for both, results and workspaces of their own."""
    pool = _pool(adapters, 5, 16, 1024, 1160)
    problems = []
    for seed, counts in ((3, [4] * 60), (9, [300, 1, 129, 0, 40])):
        x, y = _inputs(pool, sum(counts), seed=seed)
        offsets = [sum(counts[:i]) for i in range(len(counts) + 1)]
        problems.append((x, y, _int([i % 5 for i in range(len(counts))]), _int(offsets)))
    alone = [pool.add(*problem) for problem in problems]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for problem, stream in zip(problems, streams):
            with torch.cuda.stream(stream):
                got.append(pool.add(*problem))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))
    assert pool.sync_status() == 0
