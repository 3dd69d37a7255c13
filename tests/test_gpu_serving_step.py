"""GPU test of the operators of a decode step together: prompts of two requests with adapters of their own, forked
into continuations that share their pages, expert layers between, tokens sampled from the logits; step by step, and
the same step recorded once and replayed."""
import importlib
import math

import pytest
import torch

from test_gpu_attention import _int, _offsets
from test_gpu_attention_layer import _close, _weights
from test_gpu_sampling import _token

pytestmark = pytest.mark.gpu

D, HIDDEN, HEADS, KV_HEADS, VOCAB = 128, 512, 8, 2, 3001


@pytest.fixture(scope="module")
def modules(package):
    return tuple(importlib.import_module("nemotron_inference_b200." + n)
                 for n in ("attention", "attention_layer", "stack", "adapters", "sampling"))


def _pool(adapters, n, rank, inner, outer, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randn((n, rank, inner), generator=g, device="cuda") * inner ** -0.5
    b = torch.randn((n, outer, rank), generator=g, device="cuda") * 0.5 * rank ** -0.5
    return adapters.AdapterPool(a.to(torch.bfloat16), b.to(torch.bfloat16))


def _adapted(pool, x, ids, counts):
    out, start = [], 0
    for i, c in zip(ids, counts):
        rows = x[start:start + c].double()
        start += c
        a, b = pool.a[i].double(), pool.b[i].double()
        out.append((rows @ a.T) @ b.T if i >= 0 else torch.zeros((c, pool.outer), dtype=torch.float64, device="cuda"))
    return torch.cat(out)


def _expected(cache, layer, x, sequences, counts, ids, prompts):
    """The layer in 64 bits behind its bf16 projection, over what the cache holds or, for prompts, the rows' own."""
    w = layer.weights
    x64 = x.double()
    y = (x64 / torch.sqrt((x64 ** 2).mean(1, keepdim=True) + w.epsilon) * w.norm.double()).to(torch.bfloat16)
    qkv = ((y @ w.qkv.t()).double() + _adapted(layer.adapters.qkv, y, ids, counts)).unflatten(1, (-1, D))
    outs, start, p = [], 0, cache.codes.shape[4]
    for s, c in zip(sequences, counts):
        rows, n = slice(start, start + c), int(cache.lengths[s])
        start += c
        pages = cache.block_table[s, :-(-n // p)].long()
        values = cache.codes[layer.layer, pages].double() * torch.exp2(cache.exponents[layer.layer, pages].double())[..., None, None]
        k, v = values.permute(1, 0, 3, 2, 4).flatten(1, 2)[:, :n]
        if prompts:
            k, v = qkv[rows, HEADS:HEADS + KV_HEADS], qkv[rows, HEADS + KV_HEADS:]
        k, v = (t.repeat_interleave(HEADS // KV_HEADS, 1).transpose(0, 1) for t in (k, v))
        scores = qkv[rows, :HEADS].transpose(0, 1) @ k.transpose(1, 2) * D ** -0.5
        seen = torch.arange(n, device="cuda")[None] <= n - c + torch.arange(c, device="cuda")[:, None]
        outs.append((torch.softmax(scores.masked_fill(~seen, -math.inf), dim=2) @ v).transpose(0, 1).flatten(1))
    attended = torch.cat(outs)
    return x64 + attended @ w.out.double().t() + _adapted(layer.adapters.out, attended, ids, counts)


class _Model:
    def __init__(self, modules, package, synthetic):
        attention, layers, stacks, adapters, self.sampling = modules
        config = synthetic.baseline_config(max_tokens=512, experts=32, hidden=HIDDEN, routed=256, shared=512)
        self.moe = package.ExpertLayerSlice.create(config, synthetic.make_layer(config, seed=3, device="cuda").bindings)
        self.cache = attention.KvCache.allocate(2, 96, KV_HEADS, 9, 24, page_tokens=16)
        self.attention = [layers.AttentionLayer(_weights(layers, 30 + i), self.cache, i, layers.LayerAdapters(
            _pool(adapters, 3, 16, HIDDEN, (HEADS + 2 * KV_HEADS) * D, 40 + i), _pool(adapters, 3, 16, HEADS * D, HIDDEN, 50 + i)))
            for i in range(2)]
        self.order = [self.attention[0], self.moe, self.attention[1]]
        self.stack = stacks.MoeLayerStack(self.order, HIDDEN, 512)
        self.layers = layers
        g = torch.Generator(device="cuda").manual_seed(9)
        self.embedding = torch.randn((VOCAB, HIDDEN), generator=g, device="cuda")
        self.head = (torch.randn((VOCAB, HIDDEN), generator=g, device="cuda") * 2 * HIDDEN ** -0.5).to(torch.bfloat16)

    def batch(self, sequences, counts, ids, groups=None, prompts=False):
        return self.layers.TokenBatch(self.cache, _int(sequences), _offsets(counts), sum(counts), prompts,
                                      None if groups is None else _int(groups), _int(ids))

    def step(self, batch, tokens, uniform):
        """Embeddings in, the last rows' logits and the tokens sampled from them out."""
        for layer in self.attention:
            layer.batch = batch
        batch.begin()
        x = self.embedding[tokens.long()]
        hidden = torch.empty_like(x)
        self.stack.run(x, hidden)
        last = hidden[batch.offsets[1:].long() - 1]
        logits = last.to(torch.bfloat16) @ self.head.t()
        return x, logits, self.sampling.sample(logits, uniform, temperature=0.8, top_k=40, top_p=0.9)

    def check(self, batch, x, sequences, counts, ids):
        """The layers one by one; an append of the same rows changes nothing."""
        for layer in self.order:
            result = torch.empty_like(x)
            if layer is self.moe:
                layer.run_async(x, result)
            else:
                layer(x, result)
                _close(result, _expected(self.cache, layer, x, sequences, counts, ids, batch.prompts))
            x = result

    def begin(self):
        """Two prompts, and three and four continuations of them."""
        g = torch.Generator(device="cuda").manual_seed(11)
        batch = self.batch([0, 4], [200, 150], [2, -1], prompts=True)
        tokens = torch.randint(0, VOCAB, (350,), generator=g, device="cuda")
        x, _, first = self.step(batch, tokens, torch.full((2,), 0.5, device="cuda"))
        self.check(batch, x, [0, 4], [200, 150], [2, -1])
        self.cache.fork(_int([0, 0, 4, 4, 4]), _int([1, 2, 5, 6, 7]))
        return first.repeat_interleave(torch.tensor([3, 4], device="cuda"))


def test_steps_of_many_requests(modules, package, synthetic):
    sequences, counts, ids, groups = [0, 1, 2, 4, 5, 6, 7], [1] * 7, [2, 2, 0, -1, 1, 1, -1], [0, 3, 7]
    uniforms = torch.rand((6, 7), generator=torch.Generator(device="cuda").manual_seed(12), device="cuda")
    model = _Model(modules, package, synthetic)
    tokens = model.begin()
    drawn = []
    for u in uniforms:
        batch = model.batch(sequences, counts, ids, groups)
        x, logits, after = model.step(batch, tokens, u)
        assert batch.shared.tolist() == [128] * 7  # 192 tokens in full pages, and 144
        model.check(batch, x, sequences, counts, ids)
        for i in range(7):
            want, _ = _token(logits[i].float().cpu().numpy(), float(u[i]), 0.8, 40, 0.9)
            assert int(after[i]) == want
        tokens = after
        drawn.append(after.tolist())
    assert model.stack.sync_status() == 0
    assert len(set(map(tuple, zip(*drawn)))) > 2  # (the continuations have parted)

    # the same from the start, with the step recorded
    model = _Model(modules, package, synthetic)
    tokens, uniform = model.begin(), uniforms[0].clone()
    batch = model.batch(sequences, counts, ids, groups)
    again = [model.step(batch, tokens, uniform)[2].tolist()]  # (once without a graph)
    tokens.copy_(torch.tensor(again[0], device="cuda"))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, _, after = model.step(batch, tokens, uniform)
        tokens.copy_(after)
    for u in uniforms[1:]:
        uniform.copy_(u)
        graph.replay()
        again.append(tokens.tolist())
    assert again == drawn
    assert model.stack.sync_status() == 0


def test_layers_refuse_and_report(modules, package, synthetic):
    attention, layers, stacks, adapters, _ = modules
    cache = attention.KvCache.allocate(1, 40, KV_HEADS, 4, 8, page_tokens=16)
    w = _weights(layers, 1)
    qkv = _pool(adapters, 2, 8, HIDDEN, (HEADS + 2 * KV_HEADS) * D, 1)
    with pytest.raises(ValueError):
        layers.AttentionLayer(w, cache, 0, layers.LayerAdapters(out=qkv))
    layer = layers.AttentionLayer(w, cache, 0, layers.LayerAdapters(qkv=qkv))
    stack = stacks.MoeLayerStack([layer], HIDDEN, 64)
    x = torch.randn((3, HIDDEN), device="cuda")
    out, plain = torch.empty_like(x), torch.empty_like(x)
    layer.batch = layers.TokenBatch(cache, _int([0, 1]), _offsets([1, 2]), 3, groups=_int([0, 2]))
    with pytest.raises(ValueError):
        stack.run(x, out)  # `begin` has not been called
    layer.batch.begin()
    stack.run(x, plain)
    layer.batch.adapters = _int([-1, -1])  # requests without one: the same bits
    stack.run(x, out)
    assert stack.sync_status() == 0 and torch.equal(out, plain)
    layer.batch.adapters = _int([1, 7])  # one that is none
    stack.run(x, out)
    assert stack.sync_status() == 1 and stack.sync_status() == 0
    assert torch.equal(out[1:], plain[1:]) and not torch.equal(out[:1], plain[:1])
