"""GPU tests of attention over shared tokens by the kernel for more than 128 rows of queries to a group and key head.

Tolerances are those of tests/test_gpu_attention_shared.py: its kernel's weights are within 2^-11 of themselves or 2^-25 of
the largest that its reference allows (2^8), which the bounds there hold with room."""
import importlib
import random

import pytest
import torch

from test_gpu_attention import _int, _normal
from test_gpu_attention_shared import _attend, _check, _edges, _shared_cache

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
