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


def _alone(script):
    """Runs a script in a process of its own: nothing has called the operators before."""
    head = ("import importlib, sys, torch\n"
            "sys.path.insert(0, %r)\n"
            "import __graft_entry__ as entry\n"
            "package = entry.load_package()\n"
            "attention = importlib.import_module('nemotron_inference_b200.attention')\n"
            "def rows(seed, n, heads):\n"
            "    g = torch.Generator(device='cuda').manual_seed(seed)\n"
            "    return torch.randn((n, heads, 128), generator=g, device='cuda').to(torch.bfloat16)\n"
            "q, k, v = rows(1, 40, 4), rows(2, 40, 2), rows(3, 40, 2)\n"
            "offsets = torch.tensor([0, 30, 40], dtype=torch.int32, device='cuda')\n" % ROOT)
    done = subprocess.run([sys.executable, "-c", head + script], capture_output=True, text=True, timeout=300,
                          cwd=ROOT)
    assert done.returncode == 0, done.stdout[-2000:] + done.stderr[-2000:]


def test_prompts_on_a_stream_that_is_ahead_of_the_first_call():
    # the first call stands behind other work of its stream; memory that it takes held something before
    _alone("""
outs = [torch.full((40, 4, 128), 7.0, dtype=torch.bfloat16, device='cuda') for _ in range(2)]
mine = torch.zeros(1, dtype=torch.int32, device='cuda')
# (a first launch loads the kernel, which would wait for the device; it is given a word of its own)
attention._lib().nmoe_attention_prefill(0, q.data_ptr(), 512, k.data_ptr(), 256, v.data_ptr(), 256, 40, 4, 2,
                                        offsets.data_ptr(), 2, 0.1, outs[0].data_ptr(), None, mine.data_ptr())
a, b = torch.cuda.Stream(), torch.cuda.Stream()
torch.cuda.synchronize()
with torch.cuda.stream(a):
    used = [torch.full((1 << 18,), 7, dtype=torch.int32, device='cuda') for _ in range(4)]
    used += [torch.full((1,), 7, dtype=torch.int32, device='cuda') for _ in range(200)]
    torch.cuda.synchronize()
    del used
    torch.cuda._sleep(300000000)
    attention.attention_prefill(q, k, v, offsets, out=outs[0])
with torch.cuda.stream(b):
    attention.attention_prefill(q, k, v, offsets, out=outs[1])
torch.cuda.synchronize()
want = attention.attention_prefill(q, k, v, offsets)
assert attention.prefill_sync_status() == 0
assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
""")


def test_a_first_call_in_a_recording_is_refused():
    _alone("""
def recorded(call):
    graph, refused = torch.cuda.CUDAGraph(), False
    with torch.cuda.graph(graph):
        keep = torch.zeros(8, device='cuda')
        try:
            call()
        except RuntimeError as error:
            refused = 'record' in str(error)
    torch.cuda.synchronize()
    return graph, not refused
out = torch.zeros_like(q)
assert not recorded(lambda: attention.attention_prefill(q, k, v, offsets, out=out))[1]
assert not recorded(lambda: attention.KvCache.allocate(1, 4, 2, 2, 2))[1]
want = attention.attention_prefill(q, k, v, offsets)
graph, done = recorded(lambda: attention.attention_prefill(q, k, v, offsets, out=out))
assert done
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, want) and attention.prefill_sync_status() == 0
""")


def test_a_cache_makes_the_word_of_prompts_as_well():
    # (whoever records a step has its cache before)
    _alone("""
cache = attention.KvCache.allocate(1, 4, 2, 2, 2)
out = torch.zeros_like(q)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    attention.attention_prefill(q, k, v, offsets, out=out)
graph.replay()
assert attention.prefill_sync_status() == 0
assert torch.equal(out, attention.attention_prefill(q, k, v, offsets))
""")


def test_two_threads_make_one_word():
    _alone("""
import threading, time
zeros, made = torch.zeros, []
def slow(*args, **kwargs):
    made.append(args)
    time.sleep(0.2)
    return zeros(*args, **kwargs)
torch.zeros = slow
def call():
    attention.attention_prefill(q, k, v, offsets, out=torch.empty_like(q))
threads = [threading.Thread(target=call) for _ in range(4)]
for t in threads: t.start()
for t in threads: t.join()
assert len(made) == 1, made
""")


def test_a_word_of_the_callers_own(attention):
    q, k, v = (_normal(30 + i, 200, h, D).to(torch.bfloat16) for i, h in enumerate((4, 2, 2)))
    offsets = _offsets([120, 80])
    want, sums = attention.attention_prefill(q, k, v, offsets, return_lse=True)
    mine = _int([1])  # as a wait that ran out leaves it
    out, lse = attention.attention_prefill(q, k, v, offsets, return_lse=True, error=mine,
                                           out=torch.full_like(q, 7.0))
    # nothing is computed, and nothing is handed out that nobody wrote
    assert not bool(out.any()) and bool((lse == -float("inf")).all())
    assert torch.equal(attention.attention_prefill(q, k, v, offsets), want)  # others go on
    assert attention.prefill_sync_status() == 0
    assert attention.prefill_sync_status(mine) == 4 and int(mine) == 0
    out, lse = attention.attention_prefill(q, k, v, offsets, return_lse=True, error=mine)
    assert torch.equal(out, want) and torch.equal(lse, sums) and attention.prefill_sync_status(mine) == 0
    for bad in (torch.zeros(1, device="cuda"), _int([0, 0]), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            attention.attention_prefill(q, k, v, offsets, error=bad)


@pytest.mark.parametrize("heads", [4, 64])
def test_attention_does_nothing_after_books_that_failed(attention, heads):
    cache = _filled(attention, [100, 50], 2, 32, seed=9, layers=1)
    q = _normal(10, 6, heads, D).to(torch.bfloat16)
    batch = (_int([0, 1]), _offsets([4, 2]))
    want = cache.attend(0, q, *batch)
    cache.extend(_int([0]), _offsets([32 * 40]), rows=32 * 40)  # more than there are pages
    out = cache.attend(0, q, *batch, out=torch.full_like(q, 7.0))
    assert not bool(out.any())  # (of rows that have no place, no plausible results)
    assert cache.sync_status() == 6
    assert torch.equal(cache.attend(0, q, *batch), want) and cache.sync_status() == 0


@pytest.mark.parametrize("heads", [4, 64])
def test_attention_beside_a_bad_entry(attention, heads):
    cache = _filled(attention, [100, 5000, 50, 2], 2, 32, seed=9, layers=1)
    counts = [4, 3, 5, 2]
    q = _normal(10, sum(counts), heads, D).to(torch.bfloat16)
    want = cache.attend(0, q, _int([0, 1, 2, 3]), _offsets(counts))
    for place in range(4):
        sequences = [0, 1, 2, 3]
        sequences[place] = (-1, 4, 10 ** 9, -5)[place]
        got = cache.attend(0, q, _int(sequences), _offsets(counts), out=torch.full_like(q, 7.0))
        assert cache.sync_status() == 1
        rows = slice(sum(counts[:place]), sum(counts[:place + 1]))
        assert not bool(got[rows].any())
        got[rows] = want[rows]
        # (with other tiles in the batch a sequence may be cut elsewhere: the last bit of a sum)
        assert torch.allclose(got.float(), want.float(), rtol=2 ** -7, atol=2 ** -7)


def test_what_a_call_that_gave_up_left_is_cleared(attention):
    # as blocks leave it that stopped in the middle of a join: counters that are not zero
    cache = _filled(attention, [6000], 1, 64, seed=9, layers=1)
    q = _normal(10, 1, 8, D).to(torch.bfloat16)
    batch = (_int([0]), _offsets([1]))
    want = cache.attend(0, q, *batch)
    words = cache._workspace.view(torch.int32)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    counters = words[-(4096 // 4 + 128 * (D + 2) * 2 * sms):][:1024]  # (in front of the pieces)
    assert not bool(counters.any())
    counters.fill_(3)
    words[0] = 1
    assert not bool(cache.attend(0, q, *batch).any())
    assert cache.sync_status() == 4 and not bool(counters.any())
    assert torch.equal(cache.attend(0, q, *batch), want) and cache.sync_status() == 0


def test_rows_without_a_list_are_refused(attention, package):
    cache = attention.KvCache.allocate(1, 10, 2, 3, 4, 16)
    q = torch.zeros((3, 4, D), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(package.NmoeError):
        cache.attend(0, q, _int([]), _int([0]))
    with pytest.raises(package.NmoeError):
        attention.attention_prefill(q, q[:, :2], q[:, :2], _int([0]))
    assert cache.attend(0, q[:0], _int([]), _int([0])).shape == (0, 4, D)
    assert attention.attention_prefill(q[:0], q[:0, :2], q[:0, :2], _int([0])).shape == (0, 4, D)


def test_a_fork_of_a_page_that_does_not_exist(attention):
    cache = _filled(attention, [100, 0, 40], 1, 16, seed=3, layers=2)
    row = cache.block_table[0].tolist()
    row[2] = cache.block_table[0, 2] = 10 ** 6
    references = cache.references.tolist()
    page = references.index(0)
    cache.fork(_int([0]), _int([1]))
    assert cache.sync_status() == 1  # and no other page has taken its place
    assert cache.block_table[0].tolist() == row and cache.lengths.tolist() == [100, 100, 40]
    for shared in row[:2] + row[3:6]:
        references[shared] += 1
    references[page] = 1
    assert cache.references.tolist() == references
    assert cache.block_table[1].tolist() == row[:6] + [page, 0]
    bits = cache.codes.view(torch.uint8)
    assert torch.equal(bits[:, page], bits[:, row[6]])
    cache.free(_int([1]))
    assert cache.sync_status() == 0 and cache.references.tolist()[page] == 0
    cache.fork(_int([2]), _int([1]))
    assert cache.sync_status() == 0


@pytest.mark.parametrize("lengths,counts,heads,kv_heads", [
    ([20000], [1], 8, 1), ([9000, 20011], [3, 5], 8, 1), ([700] * 70, [1] * 70, 8, 1), ([30000, 5, 800], [8, 1, 2], 32, 2),
    ([2500], [300], 16, 2)])
def test_joins_that_blocks_leave(attention, lengths, counts, heads, kv_heads):
    # blocks that find pieces missing go at once, and those that bring the last ones join what is left
    cache = _filled(attention, lengths, kv_heads, 64, seed=2, layers=1)
    q = (2 * _normal(11, sum(counts), heads, D)).to(torch.bfloat16)
    batch = (_int(list(range(len(lengths)))), _offsets(counts))
    want = cache.attend(0, q, *batch, scale=0.05)
    impatient = cache._workspace.view(torch.int32)[3]
    for _ in range(10):
        impatient.fill_(1)
        assert torch.equal(cache.attend(0, q, *batch, scale=0.05, out=torch.full_like(q, 7.0)), want)
        impatient.fill_(0)
        assert torch.equal(cache.attend(0, q, *batch, scale=0.05, out=torch.full_like(q, 7.0)), want)
    assert cache.sync_status() == 0


@pytest.mark.parametrize("find", ["append", "attend"])
def test_no_row_is_written_where_no_room_was_made(attention, find):
    # a step whose append or attention finds something wrong, and the steps behind it, whose extension does nothing
    cache = _filled(attention, [40, 20], 2, 16, seed=9, layers=1)
    kv = torch.ones((2, 2, D), dtype=torch.bfloat16, device="cuda")
    q = torch.ones((2, 8, D), dtype=torch.bfloat16, device="cuda")
    bad, good = (_int([5, 1]), _offsets([1, 1])), (_int([0, 1]), _offsets([1, 1]))
    if find == "append":
        cache.append(0, kv, kv, *bad)
    else:
        cache.attend(0, q, *bad)
    codes, exponents = cache.codes.view(torch.uint8).clone(), cache.exponents.clone()
    for _ in range(2):
        cache.extend(*good, rows=2)
        cache.append(0, 3 * kv, 3 * kv, *good)
        assert not bool(cache.attend(0, q, *good).any())
    assert cache.lengths.tolist() == [40, 20]
    assert torch.equal(cache.codes.view(torch.uint8), codes) and torch.equal(cache.exponents, exponents)
    assert cache.sync_status() == 1 and cache.sync_status() == 0
    cache.extend(*good, rows=2)
    cache.append(0, kv, kv, *good)
    assert cache.sync_status() == 0 and cache.lengths.tolist() == [41, 21]
