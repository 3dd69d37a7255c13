"""CPU tests of the attention entry points: what is refused before anything reaches a device."""
import ctypes
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def attention(package):
    return importlib.import_module("nemotron_inference_b200.attention")


def _descriptor(attention, **changes):
    """A descriptor whose pointers are never followed."""
    at = 1 << 20
    fields = dict(layers=2, pages=10, kv_heads=2, page_tokens=64, max_sequences=3,
                  max_pages_per_sequence=4, codes=at, exponents=at, block_table=at, lengths=at,
                  references=at, workspace=at, workspace_bytes=1 << 30)
    fields.update(changes)
    return attention._KvCache(**fields)


def _call(attention, name, *args):
    return getattr(attention._lib(), name)(*args)


def test_workspace_bytes(attention):
    sizes = _descriptor(attention)
    small = _call(attention, "nmoe_kv_workspace_bytes", ctypes.byref(sizes))
    assert small > 0
    sizes.pages = 100000
    assert _call(attention, "nmoe_kv_workspace_bytes", ctypes.byref(sizes)) > small
    for field, value in (("layers", 0), ("pages", -1), ("kv_heads", 0), ("page_tokens", 48),
                         ("max_sequences", 0), ("max_pages_per_sequence", 2 ** 30)):
        bad = _descriptor(attention, **{field: value})
        assert _call(attention, "nmoe_kv_workspace_bytes", ctypes.byref(bad)) == 0
    assert _call(attention, "nmoe_kv_workspace_bytes", None) == 0


@pytest.mark.parametrize("changes", [
    {"codes": None}, {"codes": (1 << 20) + 64}, {"exponents": None}, {"block_table": (1 << 20) + 2},
    {"lengths": None}, {"references": None}, {"workspace": None}, {"workspace": (1 << 20) + 16},
    {"workspace_bytes": 1000}, {"page_tokens": 8}, {"pages": 0}])
def test_a_descriptor_that_is_none_is_refused_by_every_call(attention, changes):
    c = ctypes.byref(_descriptor(attention, **changes))
    p = 1 << 21
    assert _call(attention, "nmoe_kv_extend", c, None, p, p, 1, 1) == 1
    assert _call(attention, "nmoe_kv_append", c, None, 0, p, 256, p, 256, p, p, 1, 1) == 1
    assert _call(attention, "nmoe_kv_fork", c, None, p, p, 1) == 1
    assert _call(attention, "nmoe_kv_free", c, None, p, 1) == 1
    assert _call(attention, "nmoe_kv_compact", c, None) == 1
    assert _call(attention, "nmoe_kv_copy_pages", c, None, p, p, 1) == 1
    assert _call(attention, "nmoe_kv_sync_status", c, None) == 1
    assert _call(attention, "nmoe_attention_cached", c, None, 0, p, 512, 4, p, p, 1, 1, 0.1, p) == 1


def test_arguments_are_refused_before_anything_is_enqueued(attention):
    c, p = ctypes.byref(_descriptor(attention)), 1 << 21

    def cached(layer=0, q=p, stride=512, heads=4, sequences=p, offsets=p, count=1, rows=1, scale=0.1, out=p):
        return _call(attention, "nmoe_attention_cached", c, None, layer, q, stride, heads, sequences,
                     offsets, count, rows, scale, out)

    for bad in (dict(layer=2), dict(layer=-1), dict(q=None), dict(q=p + 8), dict(stride=511), dict(stride=384),
                dict(heads=3), dict(heads=0), dict(sequences=None), dict(offsets=p + 1), dict(count=-1),
                dict(rows=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(out=None), dict(out=p + 8)):
        assert cached(**bad) == 1, bad
    assert cached(rows=0) == 0 and cached(count=0) == 0  # nothing to do
    assert _call(attention, "nmoe_kv_append", c, None, 0, p, 128, p, 256, p, p, 1, 1) == 1  # rows overlap
    assert _call(attention, "nmoe_kv_fork", c, None, p, p, 4) == 1  # more than there are sequences
    assert _call(attention, "nmoe_kv_fork", c, None, p, None, 1) == 1
    assert _call(attention, "nmoe_kv_copy_pages", c, None, None, p, 1) == 1

    def prefill(q=p, k=p, tokens=8, heads=4, kv_heads=2, offsets=p, count=1, scale=0.1, out=p, error=p):
        return _call(attention, "nmoe_attention_prefill", None, q, 512, k, 256, p, 256, tokens, heads,
                     kv_heads, offsets, count, scale, out, None, error)

    for bad in (dict(q=None), dict(k=p + 2), dict(tokens=-1), dict(tokens=2 ** 31), dict(heads=5),
                dict(kv_heads=0), dict(offsets=None), dict(count=-1), dict(scale=0.0), dict(out=None),
                dict(error=None)):
        assert prefill(**bad) == 1, bad
    assert prefill(tokens=0) == 0
    assert _call(attention, "nmoe_attention_sync_status", None, None) == 1


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device behaviour")
def test_no_cpu_fallback(attention):
    q = torch.zeros((4, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention.attention_prefill(q, q, q, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(RuntimeError):
        attention.KvCache.allocate(1, 4, 1, 1, 1)
