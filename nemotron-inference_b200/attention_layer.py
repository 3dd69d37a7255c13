"""An attention layer for `MoeLayerStack`: the operators of attention.py between the projections.

The model's loop alternates expert layers with layers of other kinds
(runtime/src/api/single_token_forward_model.cpp:603-636); this is the attention kind as a caller
would write it: RMSNorm, one projection to queries, keys and values, the new rows into the cache,
attention, the projection back and the residual.  The projections are plain bf16 matrix products.

    cache = KvCache.allocate(layers=2, pages=512, kv_heads=2, max_sequences=8, max_pages_per_sequence=64)
    attention = [AttentionLayer(weights, cache, i) for i, weights in enumerate(...)]
    stack = MoeLayerStack([attention[0], moe[0], attention[1], moe[1]], hidden, max_tokens)
    batch = TokenBatch(cache, sequences, offsets, rows, prompts=True)  # prompts, then ...
    for layer in attention: layer.batch = batch
    batch.begin()
    stack.run(x, out)
    batch = TokenBatch(cache, sequences, one_each, len(sequences))     # ... a token at a time

Continuations of a prompt, forked from it, read its pages once for all of them if the batch names them as groups, and
requests can have low-rank adapters of their own beside the projections:

    layer = AttentionLayer(weights, cache, i, LayerAdapters(qkv=AdapterPool(...), out=AdapterPool(...)))
    batch = TokenBatch(cache, sequences, offsets, rows, groups=groups, adapters=ids)

`stack.sync_status()` says what a pass could not do: a batch for which there were too few pages leaves
the cache and its lengths as they were, and its results are of no use.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import rmsnorm
from .adapters import AdapterPool
from .attention import HEAD_DIM, KvCache, attention_prefill, new_error_word, prefill_sync_status


@dataclass
class TokenBatch:
    """What a pass through the stack works on: `rows` new tokens, those of sequence sequences[i] in
    rows [offsets[i], offsets[i + 1]).  `prompts`: they are whole prompts, of sequences that held
    nothing before (where one did, the cache stays as it was and its status is
    NMOE_ERR_INVALID_ARGUMENT: such rows are attended with `prompts` off).

    `groups` [n + 1]: the entries [groups[g], groups[g + 1]) continue the same tokens (`KvCache.find_shared`;
    prompts share nothing).  `adapters`: each entry's number in the layers' pools of adapters, -1 none."""
    cache: KvCache
    sequences: torch.Tensor
    offsets: torch.Tensor
    rows: int
    prompts: bool = False
    groups: Optional[torch.Tensor] = None
    adapters: Optional[torch.Tensor] = None
    shared: Optional[torch.Tensor] = None  # set by `begin`: tokens that entries have in common with their groups

    def begin(self) -> None:
        """Makes room for the new tokens, and finds what groups share, once for all layers."""
        if self.prompts:
            self.cache.require_empty(self.sequences, self.offsets)
        self.cache.extend(self.sequences, self.offsets, self.rows)
        if self.groups is not None and not self.prompts:
            self.shared = self.cache.find_shared(self.sequences, self.offsets, self.groups, out=self.shared)


@dataclass
class AttentionWeights:
    norm: torch.Tensor   # [hidden] FP32
    qkv: torch.Tensor    # [(heads + 2 kv_heads) * 128, hidden] bf16
    out: torch.Tensor    # [hidden, heads * 128] bf16
    epsilon: float = 1.0e-5


@dataclass
class LayerAdapters:
    """Adapters beside a layer's projections; None: that one has none."""
    qkv: Optional[AdapterPool] = None  # hidden -> (heads + 2 kv_heads) * 128
    out: Optional[AdapterPool] = None  # heads * 128 -> hidden


class AttentionLayer:
    def __init__(self, weights: AttentionWeights, cache: KvCache, layer: int, adapters: Optional[LayerAdapters] = None):
        total, hidden = weights.qkv.shape
        self.heads = total // HEAD_DIM - 2 * cache.kv_heads
        if total % HEAD_DIM or self.heads <= 0 or self.heads % cache.kv_heads or \
                weights.out.shape != (hidden, self.heads * HEAD_DIM) or weights.norm.shape != (hidden,):
            raise ValueError("qkv must be [(heads + 2 kv_heads) * 128, hidden], out [hidden, heads * "
                             "128], norm [hidden], with the cache's kv_heads")
        self.adapters = adapters or LayerAdapters()
        for pool, weight, name in ((self.adapters.qkv, weights.qkv, "qkv"), (self.adapters.out, weights.out, "out")):
            if pool is not None and (pool.outer, pool.inner) != tuple(weight.shape):
                raise ValueError(f"the adapters of {name} must be as wide as its projection")
        self.weights, self.cache, self.layer = weights, cache, layer
        self.batch: Optional[TokenBatch] = None
        self.error = new_error_word(cache.device)  # of this layer's prompts

    def sync_status(self) -> int:
        """Waits for the current stream; what this layer, its pools of adapters, or its cache for any layer,
        could not do, and clears it (`MoeLayerStack.sync_status` asks every layer)."""
        of_cache, of_prompts = self.cache.sync_status(), prefill_sync_status(self.error)
        of_pools = [pool.sync_status() for pool in (self.adapters.qkv, self.adapters.out) if pool is not None]
        return of_cache or of_prompts or next((status for status in of_pools if status), 0)

    def _project(self, x: torch.Tensor, weight: torch.Tensor, pool: Optional[AdapterPool]) -> torch.Tensor:
        y = x @ weight.t()
        if pool is None or self.batch.adapters is None:
            return y
        return pool.add(x, y, self.batch.adapters, self.batch.offsets, out=y)

    def __call__(self, x: torch.Tensor, out: torch.Tensor) -> None:
        """x, out: [rows, hidden] FP32 or bf16, the rows of `batch`."""
        batch, cache, w = self.batch, self.cache, self.weights
        if batch is None or batch.rows != x.shape[0]:
            raise ValueError("set `batch` to the one whose rows these are")
        if batch.groups is not None and batch.shared is None and not batch.prompts:
            raise ValueError("`begin` finds what the batch's groups share")
        y = rmsnorm(x, w.norm, w.epsilon).to(torch.bfloat16)
        qkv = self._project(y, w.qkv, self.adapters.qkv).unflatten(1, (-1, HEAD_DIM))
        q, k, v = qkv.split((self.heads, cache.kv_heads, cache.kv_heads), dim=1)
        cache.append(self.layer, k, v, batch.sequences, batch.offsets)
        if batch.prompts:
            attended = attention_prefill(q, k, v, batch.offsets, error=self.error)
        elif batch.groups is not None:
            attended = cache.attend_shared(self.layer, q, batch.sequences, batch.offsets, batch.groups, batch.shared)
        else:
            attended = cache.attend(self.layer, q, batch.sequences, batch.offsets)
        torch.add(x, self._project(attended.flatten(1), w.out, self.adapters.out), out=out)
