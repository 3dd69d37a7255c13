"""CPU tests of the entry points of a decode step for many requests: what is refused before anything reaches a
device."""
import ctypes
import importlib

import pytest
import torch

from test_attention_abi import _descriptor

P = 1 << 21  # (addresses that are never followed)


@pytest.fixture(scope="module")
def attention(package):
    return importlib.import_module("nemotron_inference_b200.attention")


@pytest.fixture(scope="module")
def adapters(package):
    return importlib.import_module("nemotron_inference_b200.adapters")


@pytest.fixture(scope="module")
def sampling(package):
    return importlib.import_module("nemotron_inference_b200.sampling")


def test_sample(sampling):
    def sample(logits=P, dtype=0, stride=100, rows=4, vocab=100, uniform=P, temperature=None, temperature_all=1.0, top_k=None,
               top_k_all=0, top_p=None, top_p_all=1.0, min_p=None, min_p_all=0.0, tokens=P, logprobs=None):
        return sampling._lib().nmoe_sample(None, logits, dtype, stride, rows, vocab, uniform, temperature, temperature_all,
                                           top_k, top_k_all, top_p, top_p_all, min_p, min_p_all, tokens, logprobs)

    nan = float("nan")
    for bad in (dict(logits=None), dict(logits=P + 2), dict(dtype=2), dict(dtype=1, logits=P + 1), dict(stride=99), dict(rows=-1),
                dict(vocab=0), dict(vocab=-5), dict(uniform=None), dict(uniform=P + 1), dict(temperature=P + 2),
                dict(temperature_all=nan), dict(top_k=P + 1), dict(top_p=P + 3), dict(top_p_all=nan), dict(min_p=P + 2),
                dict(min_p_all=nan), dict(tokens=None), dict(tokens=P + 2), dict(logprobs=P + 1), dict(rows=2 ** 40)):
        assert sample(**bad) == 1, bad
    assert sample(vocab=393217, stride=393217) == 3 and sample(dtype=1, vocab=786433, stride=786433) == 3  # beyond a row's size
    assert sample(rows=0) == 0


def test_attention_shared(attention):
    lib = attention._lib()
    c = ctypes.byref(_descriptor(attention))
    needed = lib.nmoe_attention_shared_workspace_bytes(3, 4)
    assert needed > 0 and lib.nmoe_attention_shared_workspace_bytes(300, 4) > needed
    for rows, heads in ((0, 4), (-1, 4), (3, 0), (3, 70000), (2 ** 40, 4)):
        assert lib.nmoe_attention_shared_workspace_bytes(rows, heads) == 0

    def shared(cache=c, layer=0, q=P, stride=512, heads=4, sequences=P, offsets=P, count=3, rows=3, groups=P, group_count=1, plan=P,
               scale=0.1, workspace=P, size=needed, out=P):
        return lib.nmoe_attention_shared(cache, None, layer, q, stride, heads, sequences, offsets, count, rows, groups, group_count,
                                         plan, scale, workspace, size, out)

    for bad in (dict(cache=None), dict(layer=2), dict(q=None), dict(q=P + 8), dict(stride=384), dict(heads=3), dict(sequences=None),
                dict(offsets=P + 2), dict(count=-1), dict(rows=-1), dict(groups=None), dict(groups=P + 1), dict(group_count=-1),
                dict(group_count=4), dict(plan=None), dict(plan=P + 2), dict(scale=0.0), dict(workspace=None),
                dict(workspace=P + 128), dict(size=needed - 1), dict(out=None), dict(out=P + 8),
                dict(cache=ctypes.byref(_descriptor(attention, page_tokens=8)))):
        assert shared(**bad) == 1, bad
    assert shared(rows=0) == 0 and shared(count=0, group_count=0) == 0

    def find(cache=c, sequences=P, offsets=P, count=3, rows=3, groups=P, group_count=1, plan=P):
        return lib.nmoe_kv_find_shared(cache, None, sequences, offsets, count, rows, groups, group_count, plan)

    for bad in (dict(cache=None), dict(sequences=None), dict(offsets=None), dict(count=-1), dict(rows=-1), dict(groups=None),
                dict(group_count=4), dict(group_count=-1), dict(groups=P + 2), dict(plan=None), dict(plan=P + 1)):
        assert find(**bad) == 1, bad
    assert find(count=0, group_count=0) == 0


def test_adapters(adapters):
    lib = adapters._lib()

    def pool(**changes):
        fields = dict(adapters=3, rank=16, inner=64, outer=128, a=P, b=P, scales=P)
        fields.update(changes)
        return ctypes.byref(adapters._Adapters(**fields))

    needed = lib.nmoe_adapters_workspace_bytes(pool(), 10, 2)
    assert needed >= 10 * 16 * 4

    def add(p=None, x=P, x_stride=64, y=P, y_stride=128, out=P, out_stride=128, rows=10, ids=P, offsets=P, count=2, workspace=P,
            size=needed, error=P):
        return lib.nmoe_adapters_add(p or pool(), None, x, x_stride, y, y_stride, out, out_stride, rows, ids, offsets, count, workspace,
                                     size, error)

    for change in (dict(adapters=0), dict(rank=0), dict(rank=12), dict(rank=136), dict(inner=60), dict(outer=4), dict(inner=0),
                   dict(adapters=2 ** 30)):
        assert add(pool(**change)) == 1 and lib.nmoe_adapters_workspace_bytes(pool(**change), 10, 2) == 0, change
    for change in (dict(a=None), dict(b=P + 8), dict(scales=None), dict(scales=P + 2)):
        assert add(pool(**change)) == 1, change
    for bad in (dict(x=None), dict(x=P + 8), dict(x_stride=56), dict(x_stride=65), dict(y=None), dict(y_stride=120), dict(out=None),
                dict(out_stride=132), dict(rows=-1), dict(rows=2 ** 30), dict(ids=None), dict(offsets=None), dict(offsets=P + 2),
                dict(count=-1), dict(workspace=None), dict(workspace=P + 64), dict(size=needed - 1), dict(error=None),
                dict(error=P + 2)):
        assert add(**bad) == 1, bad
    assert add(rows=0) == 0 and add(count=0) == 0
    assert lib.nmoe_adapters_workspace_bytes(None, 10, 2) == 0 and lib.nmoe_adapters_workspace_bytes(pool(), 0, 2) == 0
    assert lib.nmoe_adapters_sync_status(None, None) == 1


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device behaviour")
def test_no_cpu_fallback(adapters, sampling):
    with pytest.raises(ValueError):
        sampling.sample(torch.zeros((2, 10)), torch.zeros(2))
    with pytest.raises(ValueError):
        adapters.AdapterPool(torch.zeros((1, 8, 64), dtype=torch.bfloat16), torch.zeros((1, 64, 8), dtype=torch.bfloat16))
