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

`stack.sync_status()` says what a pass could not do: a batch for which there were too few pages leaves
the cache and its lengths as they were, and its results are of no use.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import rmsnorm
from .attention import HEAD_DIM, KvCache, attention_prefill, new_error_word, prefill_sync_status


@dataclass
class TokenBatch:
    """What a pass through the stack works on: `rows` new tokens, those of sequence sequences[i] in
    rows [offsets[i], offsets[i + 1]).  `prompts`: they are whole prompts, of sequences that held
    nothing before (where one did, the cache stays as it was and its status is
    NMOE_ERR_INVALID_ARGUMENT: such rows are attended with `prompts` off)."""
    cache: KvCache
    sequences: torch.Tensor
    offsets: torch.Tensor
    rows: int
    prompts: bool = False

    def begin(self) -> None:
        """Makes room for the new tokens, once for all layers."""
        if self.prompts:
            self.cache.require_empty(self.sequences, self.offsets)
        self.cache.extend(self.sequences, self.offsets, self.rows)


@dataclass
class AttentionWeights:
    norm: torch.Tensor   # [hidden] FP32
    qkv: torch.Tensor    # [(heads + 2 kv_heads) * 128, hidden] bf16
    out: torch.Tensor    # [hidden, heads * 128] bf16
    epsilon: float = 1.0e-5


class AttentionLayer:
    def __init__(self, weights: AttentionWeights, cache: KvCache, layer: int):
        total, hidden = weights.qkv.shape
        self.heads = total // HEAD_DIM - 2 * cache.kv_heads
        if total % HEAD_DIM or self.heads <= 0 or self.heads % cache.kv_heads or \
                weights.out.shape != (hidden, self.heads * HEAD_DIM) or weights.norm.shape != (hidden,):
            raise ValueError("qkv must be [(heads + 2 kv_heads) * 128, hidden], out [hidden, heads * "
                             "128], norm [hidden], with the cache's kv_heads")
        self.weights, self.cache, self.layer = weights, cache, layer
        self.batch: Optional[TokenBatch] = None
        self.error = new_error_word(cache.device)  # of this layer's prompts

    def sync_status(self) -> int:
        """Waits for the current stream; what this layer, or its cache for any layer, could not do, and
        clears it (`MoeLayerStack.sync_status` asks every layer)."""
        of_cache, of_prompts = self.cache.sync_status(), prefill_sync_status(self.error)
        return of_cache or of_prompts

    def __call__(self, x: torch.Tensor, out: torch.Tensor) -> None:
        """x, out: [rows, hidden] FP32 or bf16, the rows of `batch`."""
        batch, cache, w = self.batch, self.cache, self.weights
        if batch is None or batch.rows != x.shape[0]:
            raise ValueError("set `batch` to the one whose rows these are")
        y = rmsnorm(x, w.norm, w.epsilon).to(torch.bfloat16)
        qkv = (y @ w.qkv.t()).unflatten(1, (-1, HEAD_DIM))
        q, k, v = qkv.split((self.heads, cache.kv_heads, cache.kv_heads), dim=1)
        cache.append(self.layer, k, v, batch.sequences, batch.offsets)
        if batch.prompts:
            attended = attention_prefill(q, k, v, batch.offsets, error=self.error)
        else:
            attended = cache.attend(self.layer, q, batch.sequences, batch.offsets)
        torch.add(x, attended.flatten(1) @ w.out.t(), out=out)
