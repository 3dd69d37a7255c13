"""GPU test of attention layers between expert layers in one stack: prompts, then tokens one at a
time, then two continuations of a prompt."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D, HIDDEN, HEADS, KV_HEADS = 128, 512, 8, 2


@pytest.fixture(scope="module")
def modules(package):
    return tuple(importlib.import_module("nemotron_inference_b200." + n)
                 for n in ("attention", "attention_layer", "stack"))


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _weights(layers, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda") / math.sqrt(shape[-1])

    return layers.AttentionWeights(
        norm=1 + 0.1 * torch.randn((HIDDEN,), generator=g, device="cuda"),
        qkv=normal((HEADS + 2 * KV_HEADS) * D, HIDDEN).to(torch.bfloat16),
        out=normal(HIDDEN, HEADS * D).to(torch.bfloat16))


def _expected(cache, layer, weights, x, sequences, counts, keys_of_the_prompt):
    """The layer in 64 bits behind its bf16 projection, over what the cache holds or, for prompts,
    the rows' own keys and values."""
    x64 = x.double()
    y = x64 / torch.sqrt((x64 ** 2).mean(1, keepdim=True) + weights.epsilon) * weights.norm.double()
    qkv = (y.to(torch.bfloat16) @ weights.qkv.t()).double().unflatten(1, (-1, D))
    outs, start, p = [], 0, cache.codes.shape[4]
    for s, c in zip(sequences, counts):
        rows = slice(start, start + c)
        n = int(cache.lengths[s])
        if keys_of_the_prompt:
            k, v = qkv[rows, HEADS:HEADS + KV_HEADS], qkv[rows, HEADS + KV_HEADS:]
        else:
            pages = cache.block_table[s, :-(-n // p)].long()
            values = cache.codes[layer, pages].double() * torch.exp2(
                cache.exponents[layer, pages].double())[..., None, None]
            k, v = values.permute(1, 0, 3, 2, 4).flatten(1, 2)[:, :n]
        k, v = (t.repeat_interleave(HEADS // KV_HEADS, 1).transpose(0, 1) for t in (k, v))
        scores = qkv[rows, :HEADS].transpose(0, 1) @ k.transpose(1, 2) * D ** -0.5
        seen = torch.arange(n, device="cuda")[None] <= n - c + torch.arange(c, device="cuda")[:, None]
        w = torch.softmax(scores.masked_fill(~seen, -math.inf), dim=2)
        outs.append((w @ v).transpose(0, 1).flatten(1))
        start += c
    return x64 + torch.cat(outs) @ weights.out.double().t()


def _close(got, want):
    # the layer's own part (want - x) has a size of about one; of its steps in bf16 the attended rows
    # (2^-8 each of 1024 terms) and their product's result (2^-8) are the coarsest: 2^-8 of the rms
    # each, four times that for the largest of some thousand values, and a flip of the normalised rows'
    # rounding to bf16 as much again
    error = (got.double() - want).abs().max()
    assert float(error) <= 12 * 2 ** -8 * max(1.0, float(want.abs().max()) / 4)


def test_stack_of_attention_and_expert_layers(modules, package, synthetic):
    attention, layers, stacks = modules
    config = synthetic.baseline_config(max_tokens=256, experts=32, hidden=HIDDEN, routed=256, shared=512)
    moe = [package.ExpertLayerSlice.create(config, synthetic.make_layer(config, seed=i, device="cuda").bindings)
           for i in range(2)]
    cache = attention.KvCache.allocate(2, 64, KV_HEADS, 6, 20, page_tokens=16)
    weights = [_weights(layers, 30 + i) for i in range(2)]
    mine = [layers.AttentionLayer(w, cache, i) for i, w in enumerate(weights)]
    order = [mine[0], moe[0], mine[1], moe[1]]
    stack = stacks.MoeLayerStack(order, HIDDEN, 256)
    g = torch.Generator(device="cuda").manual_seed(5)

    def run(sequences, counts, prompts):
        offsets = [0]
        for c in counts:
            offsets.append(offsets[-1] + c)
        rows = offsets[-1]
        x = torch.randn((rows, HIDDEN), generator=g, device="cuda")
        batch = layers.TokenBatch(cache, _int(sequences), _int(offsets), rows, prompts)
        for layer in mine:
            layer.batch = batch
        batch.begin()
        got = torch.empty_like(x)
        stack.run(x, got)
        # the same layers one by one; an append of the same rows changes nothing
        current = x
        for layer in order:
            result = torch.empty_like(x)
            if layer in mine:
                layer(current, result)
                _close(result, _expected(cache, layer.layer, weights[layer.layer], current, sequences,
                                         counts, prompts))
            else:
                layer.run_async(current, result)
            current = result
        assert torch.equal(got, current)
        assert cache.sync_status() == 0 and attention.prefill_sync_status() == 0
        assert all(layer.sync_status() == 0 for layer in moe)

    run([0, 3, 4], [70, 1, 33], prompts=True)
    for _ in range(3):
        run([4, 0, 3], [1, 1, 1], prompts=False)
    cache.fork(_int([0, 0]), _int([1, 2]))
    run([0, 1, 2], [1, 3, 1], prompts=False)  # (one of them verifies drafted tokens)
    cache.free(_int([0, 3]))
    cache.compact()
    run([1, 2, 4], [2, 1, 1], prompts=False)
    assert cache.lengths.tolist() == [0, 78, 75, 0, 37, 0]


def test_attention_layer_refusals(modules):
    attention, layers, _ = modules
    cache = attention.KvCache.allocate(1, 4, KV_HEADS, 2, 2)
    w = _weights(layers, 1)
    with pytest.raises(ValueError):
        layers.AttentionLayer(layers.AttentionWeights(w.norm, w.qkv[:-1], w.out), cache, 0)
    layer = layers.AttentionLayer(w, cache, 0)
    x = torch.zeros((2, HIDDEN), device="cuda")
    with pytest.raises(ValueError):
        layer(x, torch.empty_like(x))  # no batch
    layer.batch = layers.TokenBatch(cache, _int([0]), _int([0, 1]), 1)
    with pytest.raises(ValueError):
        layer(x, torch.empty_like(x))  # another one's rows


def _layer(modules, cache):
    attention, layers, stacks = modules
    layer = layers.AttentionLayer(_weights(layers, 1), cache, 0)
    return layer, stacks.MoeLayerStack([layer], HIDDEN, 64)


def _batch(modules, layer, sequences, counts, prompts=False):
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    layer.batch = modules[1].TokenBatch(layer.cache, _int(sequences), _int(offsets), offsets[-1], prompts)
    layer.batch.begin()
    x = torch.randn((offsets[-1], HIDDEN), device="cuda")
    return x, torch.empty_like(x)


def test_a_stack_reports_what_its_cache_could_not_do(modules):
    attention = modules[0]
    cache = attention.KvCache.allocate(1, 4, KV_HEADS, 2, 4, page_tokens=16)
    layer, stack = _layer(modules, cache)
    stack.run(*_batch(modules, layer, [0], [40], prompts=True))
    assert stack.sync_status() == 0
    x, out = _batch(modules, layer, [0, 1], [1, 30])  # two more pages, of which there is one
    stack.run(x, out)
    assert stack.sync_status() == 6 and cache.lengths.tolist() == [40, 0]
    assert torch.equal(out, x)  # (no attended rows were added)
    stack.run(*_batch(modules, layer, [0], [1]))
    assert stack.sync_status() == 0 and cache.lengths.tolist() == [41, 0]


def test_a_stack_reports_a_wait_of_its_prompts_that_ran_out(modules):
    attention = modules[0]
    cache = attention.KvCache.allocate(1, 8, KV_HEADS, 2, 4, page_tokens=16)
    layer, stack = _layer(modules, cache)
    layer.error.fill_(1)  # as the kernel leaves it
    stack.run(*_batch(modules, layer, [0], [20], prompts=True))
    assert attention.prefill_sync_status() == 0  # (another one's)
    assert stack.sync_status() == 4 and stack.sync_status() == 0


def test_whole_prompts_of_sequences_that_hold_tokens_are_refused(modules):
    attention = modules[0]
    cache = attention.KvCache.allocate(1, 16, KV_HEADS, 4, 4, page_tokens=16)
    layer, stack = _layer(modules, cache)
    stack.run(*_batch(modules, layer, [0, 2], [20, 5], prompts=True))
    assert stack.sync_status() == 0
    codes = cache.codes.view(torch.uint8).clone()
    for sequences, counts in (([1, 0], [3, 4]), ([2], [1]), ([0, 1], [1, 0])):
        stack.run(*_batch(modules, layer, sequences, counts, prompts=True))
        assert stack.sync_status() == 1
        assert cache.lengths.tolist() == [20, 0, 5, 0] and torch.equal(cache.codes.view(torch.uint8), codes)
    # no rows for it: nothing of it is left out; a list that names what is not there is the books' to refuse
    stack.run(*_batch(modules, layer, [0, 1], [0, 7], prompts=True))
    assert stack.sync_status() == 0 and cache.lengths.tolist() == [20, 7, 5, 0]
    stack.run(*_batch(modules, layer, [9, -1], [2, 3], prompts=True))
    assert stack.sync_status() == 1 and cache.lengths.tolist() == [20, 7, 5, 0]
