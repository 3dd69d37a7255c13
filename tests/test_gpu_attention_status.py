"""GPU tests of what the attention operators do when something is wrong: lists that name what is not
there, pools that are full, status words that were never made or are still set."""
import importlib
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_attention import _append_model, _filled, _int, _normal, _offsets

pytestmark = pytest.mark.gpu

D = 128
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def attention(package):
    return importlib.import_module("nemotron_inference_b200.attention")


@pytest.mark.parametrize("kv_heads", [1, 3])
@pytest.mark.parametrize("bad", ["sequence", "rows", "page"])
def test_append_beside_a_bad_entry_writes_all_others(attention, kv_heads, bad):
    # many sequences whose last pages are begun and get larger values; the bad entry stands in front, in
    # the middle and at the end of the list
    p, n = 16, 80
    held = [(7 * i) % 50 + 1 for i in range(n)]
    counts = [(3 * i) % 9 + 1 for i in range(n)]
    lengths, rows = [h + c for h, c in zip(held, counts)], sum(counts)
    kv = (_normal(22, rows, 2, kv_heads, D) * 8).to(torch.bfloat16)
    k, v = kv[:, 0], kv[:, 1]
    cache = _filled(attention, lengths, kv_heads, p, seed=21)
    codes, exponents = _append_model(cache, 1, k, v, list(range(n)), counts)
    for place in (0, n // 2, n - 1):
        cache = _filled(attention, lengths, kv_heads, p, seed=21)
        mine = torch.zeros_like(cache.exponents, dtype=torch.bool)
        for i in set(range(n)) - {place}:
            mine[:, cache.block_table[i, :-(-lengths[i] // p)].long()] = True
        sequences = list(range(n))
        if bad == "sequence":
            sequences[place] = n + 5
        elif bad == "rows":
            cache.lengths[place] = counts[place] - 1
        else:
            cache.block_table[place, held[place] // p:] = 10 ** 6
        cache.append(1, k, v, _int(sequences), _offsets(counts))
        assert cache.sync_status() == 1
        assert torch.equal(cache.exponents[mine], exponents[mine])
        got = cache.codes.double()
        same = (got == codes) | (got.isnan() & codes.isnan())
        assert bool(same[mine].all())


def test_what_an_append_finds_wrong_keeps_the_books_as_they_are(attention):
    cache = _filled(attention, [100, 50, 30], 2, 32, seed=9)
    before = [t.clone() for t in (cache.block_table, cache.lengths, cache.references)]
    kv = torch.ones((1, 2, D), dtype=torch.bfloat16, device="cuda")
    cache.append(0, kv, kv, _int([7]), _offsets([1]))
    cache.extend(_int([0]), _offsets([1]), rows=1)
    cache.free(_int([1]))
    cache.fork(_int([0]), _int([2]))
    cache.compact()
    assert cache.sync_status() == 1
    for a, b in zip(before, (cache.block_table, cache.lengths, cache.references)):
        assert torch.equal(a, b)
    cache.free(_int([1]))
    assert cache.sync_status() == 0 and cache.lengths.tolist() == [100, 0, 30]
