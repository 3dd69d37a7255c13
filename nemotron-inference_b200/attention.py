"""Attention over prompts and over a paged 8-bit cache of keys and values.

The attention layers between the expert layers of a model are the caller's own code
(runtime/src/api/single_token_forward_model.cpp:603-636); these are the operators such a
layer runs between its projections, over the C ABI of include/nmoe.h:

    cache = KvCache.allocate(layers, pages, kv_heads, max_sequences, max_pages_per_sequence)
    cache.extend(sequences, offsets)                  # once a step: room for the new tokens
    for every attention layer:
        cache.append(layer, k, v, sequences, offsets)     # the new rows, as 8-bit codes
        out = attention_prefill(q, k, v, offsets)         # whole prompts, or
        out = cache.attend(layer, q, sequences, offsets)  # new rows over all tokens so far
        out = cache.attend_shared(layer, q, sequences, offsets, groups, shared)  # the same, or
                                                          # continuations of a prompt together
    cache.fork(parents, children)                     # several continuations of a prompt
    cache.free(sequences)                             # finished
    cache.compact()                                   # the pages in use, without holes

q is [rows, heads, 128] bf16, k and v [rows, kv_heads, 128]; slices of a fused projection's
rows are taken as they lie.  `sequences` [n] (rows of the block table, each at most once) and
`offsets` [n + 1] (rows of each) are int32 tensors on the device; the host reads neither, so
a step can be recorded in a CUDA graph; what a call keeps on the device (a cache's workspace, the
word of `attention_prefill`) is made before that, by a `KvCache` or a call that is not recorded.
Calls run on the current stream; a cache is used by one stream at a time.
"""
from __future__ import annotations

import ctypes
import threading
from typing import Dict, Optional

import torch

from . import NMOE_OK, NmoeError, _check, _stream, load_library

HEAD_DIM = 128
DEFAULT_SCALE = HEAD_DIM ** -0.5
_MOST_ROWS = 2 ** 30 - 1
_BAD_SEQUENCE = 17  # kCacheBadSequence of csrc/attention.h


class _KvCache(ctypes.Structure):
    _fields_ = [("layers", ctypes.c_int32), ("pages", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("page_tokens", ctypes.c_int32),
                ("max_sequences", ctypes.c_int32), ("max_pages_per_sequence", ctypes.c_int32),
                ("codes", ctypes.c_void_p), ("exponents", ctypes.c_void_p),
                ("block_table", ctypes.c_void_p), ("lengths", ctypes.c_void_p),
                ("references", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_size_t)]


_library = None


def _lib() -> ctypes.CDLL:
    global _library
    if _library is None:
        lib = load_library()
        vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
        cache = ctypes.POINTER(_KvCache)
        lib.nmoe_kv_workspace_bytes.restype = ctypes.c_size_t
        lib.nmoe_kv_workspace_bytes.argtypes = [cache]
        lib.nmoe_kv_extend.argtypes = [cache, vp, vp, vp, i32, i64]
        lib.nmoe_kv_append.argtypes = [cache, vp, i32, vp, i64, vp, i64, vp, vp, i32, i64]
        lib.nmoe_kv_fork.argtypes = [cache, vp, vp, vp, i32]
        lib.nmoe_kv_free.argtypes = [cache, vp, vp, i32]
        lib.nmoe_kv_compact.argtypes = [cache, vp]
        lib.nmoe_kv_copy_pages.argtypes = [cache, vp, vp, vp, i32]
        lib.nmoe_kv_sync_status.argtypes = [cache, vp]
        lib.nmoe_attention_cached.argtypes = [cache, vp, i32, vp, i64, i32, vp, vp, i32, i64, f32, vp]
        lib.nmoe_kv_find_shared.argtypes = [cache, vp, vp, vp, i32, i64, vp, i32, vp]
        lib.nmoe_attention_shared_workspace_bytes.restype = ctypes.c_size_t
        lib.nmoe_attention_shared_workspace_bytes.argtypes = [i64, i32]
        lib.nmoe_attention_shared.argtypes = [cache, vp, i32, vp, i64, i32, vp, vp, i32, i64, vp, i32, vp, f32,
                                              vp, ctypes.c_size_t, vp]
        lib.nmoe_attention_prefill.argtypes = [vp, vp, i64, vp, i64, vp, i64, i64, i32, i32, vp, i32,
                                               f32, vp, vp, vp]
        lib.nmoe_attention_sync_status.argtypes = [vp, vp]
        _library = lib
    return _library


def _row_layout(t: torch.Tensor, name: str, device: torch.device):
    """Rows, heads and the elements from row to row of a [rows, heads, 128] bf16 tensor whose rows have
    their heads side by side (rows may lie further apart)."""
    shape, stride = t.shape, t.stride()
    if t.dtype is torch.bfloat16 and len(shape) == 3 and t.device == device:
        rows, heads, dim = shape
        if dim == HEAD_DIM and heads and (
                not rows or (stride[2] == 1 and (heads == 1 or stride[1] == HEAD_DIM))):
            return rows, heads, stride[0] if rows > 1 else heads * HEAD_DIM
    if t.device != device:
        raise ValueError(f"{name} must be on {device}: this library has no CPU path")
    if t.dtype is not torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, not {t.dtype}")
    if len(shape) != 3 or shape[2] != HEAD_DIM or shape[1] == 0:
        raise ValueError(f"{name} must be [rows, heads, {HEAD_DIM}], not {list(shape)}")
    raise ValueError(f"{name}: the heads of a row must lie side by side")


def _require_list(t: torch.Tensor, name: str, device: torch.device) -> None:
    if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous int32 vector on {device}")


def _require_word(t: torch.Tensor, device: torch.device) -> None:
    if t.dtype is not torch.int32 or t.numel() != 1 or t.device != device:
        raise ValueError(f"error must be one int32 on {device}")


def _stream_of(device: torch.device, what: str) -> int:
    """The current stream, if `device` is the current device."""
    if device.type != "cuda":
        raise ValueError(f"{what} must be a CUDA tensor: this library has no CPU path")
    index = device.index
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"{what} is on {device}, which is not the current device")
    return torch._C._cuda_getCurrentRawStream(index)


def _output(out: Optional[torch.Tensor], q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype != torch.bfloat16 or out.device != q.device or \
            not out.is_contiguous():
        raise ValueError(f"out must be contiguous bfloat16 {list(q.shape)} on {q.device}")
    return out


def _zeros(elements: int, dtype: torch.dtype, device: torch.device, what: str) -> torch.Tensor:
    """Memory that every stream finds zero: the fill is over when this returns, and no node of a graph."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} is made before anything that uses it is recorded in a CUDA graph")
    made = torch.zeros(elements, dtype=dtype, device=device)
    torch.cuda.current_stream(device).synchronize()
    return made


def new_error_word(device: torch.device) -> torch.Tensor:
    """A word for `attention_prefill`."""
    return _zeros(1, torch.int32, device, "the word of attention_prefill")


_error_words: Dict[int, torch.Tensor] = {}
_error_words_lock = threading.Lock()


def _error_word(device: torch.device) -> torch.Tensor:
    """The word of the calls of `attention_prefill` on a device that are given none."""
    error = _error_words.get(device.index)
    if error is None:
        with _error_words_lock:
            error = _error_words.get(device.index)
            if error is None:
                error = _error_words[device.index] = new_error_word(device)
    return error


def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
                      scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                      return_lse: bool = False, error: Optional[torch.Tensor] = None):
    """Causal attention over whole prompts packed one behind the other: prompt i is the rows
    [offsets[i], offsets[i + 1]), and each of its rows sees those up to itself.  Query head h
    attends key head h // (heads // kv_heads).  Returns [rows, heads, 128] bf16 and, if asked
    for, the FP32 logarithms [rows, heads] of the rows' sums of exponentials.  Rows of no prompt
    are as `out` had them, undefined without it.  `scale` is 1 / sqrt(128) unless given.

    `error`: an int32 word on the device, zero at first (`new_error_word`), in which a call whose
    waits run out leaves a status; calls compute nothing while it holds one
    (`prefill_sync_status`).  Without it all calls on a device have one word together: streams or
    models that should not stop each other are given words of their own."""
    device = q.device
    stream = _stream_of(device, "q")
    rows, heads, q_stride = _row_layout(q, "q", device)
    k_rows, kv_heads, k_stride = _row_layout(k, "k", device)
    v_rows, v_heads, v_stride = _row_layout(v, "v", device)
    _require_list(offsets, "offsets", device)
    prompts = offsets.shape[0] - 1
    if k_rows != rows or v_rows != rows or v_heads != kv_heads or heads % kv_heads or prompts < (rows > 0):
        raise NmoeError(1, "attention_prefill", "k and v need q's rows and a divisor of its heads, "
                                                "offsets one entry more than there are prompts, rows a prompt")
    out = _output(out, q)
    lse = q.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
    if error is None:
        error = _error_words.get(device.index)
        if error is None:
            error = _error_word(device)
    else:
        _require_word(error, device)
    _check((_library or _lib()).nmoe_attention_prefill(
        stream, q.data_ptr(), q_stride, k.data_ptr(), k_stride, v.data_ptr(), v_stride, rows, heads,
        kv_heads, offsets.data_ptr(), prompts, DEFAULT_SCALE if scale is None else scale,
        out.data_ptr(), None if lse is None else lse.data_ptr(), error.data_ptr()),
        "nmoe_attention_prefill")
    return (out, lse) if return_lse else out


def prefill_sync_status(error: Optional[torch.Tensor] = None) -> int:
    """Waits for the current stream; what calls of `attention_prefill` with this word, or with none on
    this device, could not do, and clears it."""
    if error is None:
        error = _error_words.get(torch.cuda.current_device())
    else:
        _require_word(error, torch.device("cuda", torch.cuda.current_device()))
    return NMOE_OK if error is None else _lib().nmoe_attention_sync_status(error.data_ptr(), _stream())


class KvCache:
    """Keys and values of `layers` attention layers in pages of `page_tokens` tokens: E4M3 codes
    with an exponent for each page, head, and keys or values (`nmoe_kv_cache`, include/nmoe.h).
    The tensors are the caller's and may be read or set between calls."""

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, block_table: torch.Tensor,
                 lengths: torch.Tensor, references: torch.Tensor):
        """codes [layers, pages, 2, kv_heads, page_tokens, 128] float8_e4m3fn, exponents
        [layers, pages, 2, kv_heads] int8, block_table [max_sequences, max_pages] int32, lengths
        [max_sequences] int32, references [pages] int32."""
        device = codes.device
        _stream_of(device, "codes")
        if codes.dtype != torch.float8_e4m3fn or codes.dim() != 6 or codes.shape[2] != 2 or \
                codes.shape[5] != HEAD_DIM:
            raise ValueError("codes must be float8_e4m3fn [layers, pages, 2, kv_heads, page_tokens, "
                             f"{HEAD_DIM}]")
        if codes.shape[4] not in (16, 32, 64, 128):
            raise ValueError("page_tokens must be 16, 32, 64 or 128")
        for t, name, dtype, shape in (
                (exponents, "exponents", torch.int8, codes.shape[:4]),
                (block_table, "block_table", torch.int32, block_table.shape),
                (lengths, "lengths", torch.int32, block_table.shape[:1]),
                (references, "references", torch.int32, codes.shape[1:2])):
            if t.dtype != dtype or t.shape != shape or t.device != device:
                raise ValueError(f"{name} must be {dtype} {list(shape)} on {device}")
        if block_table.dim() != 2:
            raise ValueError("block_table must be [max_sequences, max_pages]")
        for t in (codes, exponents, block_table, lengths, references):
            if not t.is_contiguous():
                raise ValueError("the cache's tensors must be contiguous")
        self.codes, self.exponents = codes, exponents
        self.block_table, self.lengths, self.references = block_table, lengths, references
        self.device, self.kv_heads = device, codes.shape[3]
        self._c = _KvCache(codes.shape[0], codes.shape[1], codes.shape[3], codes.shape[4],
                           block_table.shape[0], block_table.shape[1], codes.data_ptr(),
                           exponents.data_ptr(), block_table.data_ptr(), lengths.data_ptr(),
                           references.data_ptr(), None, 0)
        needed = _lib().nmoe_kv_workspace_bytes(ctypes.byref(self._c))
        if needed == 0:
            raise NmoeError(1, "KvCache", "a size is zero or too large")
        self._workspace = _zeros(needed, torch.uint8, device, "a cache's workspace")
        self._error = self._workspace[:4].view(torch.int32)  # what the books go by
        self._c.workspace, self._c.workspace_bytes = self._workspace.data_ptr(), needed
        self._ref = ctypes.byref(self._c)
        _error_word(device)  # (what records a step with a cache may begin with prompts)

    @staticmethod
    def allocate(layers: int, pages: int, kv_heads: int, max_sequences: int,
                 max_pages_per_sequence: int, page_tokens: int = 64, device=None) -> "KvCache":
        """An empty cache on the current device."""
        if not torch.cuda.is_available():
            raise RuntimeError("KvCache needs a CUDA device: there is no CPU path")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a cache is made before anything that uses it is recorded in a CUDA graph")
        device = device or torch.device("cuda", torch.cuda.current_device())
        int32 = dict(dtype=torch.int32, device=device)
        codes = torch.zeros((layers, pages, 2, kv_heads, page_tokens, HEAD_DIM), dtype=torch.uint8,
                            device=device).view(torch.float8_e4m3fn)
        exponents = torch.zeros((layers, pages, 2, kv_heads), dtype=torch.int8, device=device)
        return KvCache(codes, exponents, torch.zeros((max_sequences, max_pages_per_sequence), **int32),
                       torch.zeros((max_sequences,), **int32), torch.zeros((pages,), **int32))

    def _batch(self, sequences: torch.Tensor, offsets: torch.Tensor) -> int:
        """The current stream, if the lists are a batch's."""
        device = self.device
        _require_list(sequences, "sequences", device)
        _require_list(offsets, "offsets", device)
        if offsets.shape[0] != sequences.shape[0] + 1:
            raise ValueError("offsets must have one entry more than sequences")
        return _stream_of(device, "the cache")

    def extend(self, sequences: torch.Tensor, offsets: torch.Tensor, rows: int) -> None:
        """Makes room for `rows` new tokens, entry i's offsets[i + 1] - offsets[i] of them: the
        lowest free pages, in list order.  Too few: NMOE_ERR_CAPACITY from `sync_status`, and
        nothing has changed."""
        stream = self._batch(sequences, offsets)
        _check(_lib().nmoe_kv_extend(self._ref, stream, sequences.data_ptr(), offsets.data_ptr(),
                                     sequences.numel(), rows), "nmoe_kv_extend")

    def require_empty(self, sequences: torch.Tensor, offsets: torch.Tensor) -> None:
        """NMOE_ERR_INVALID_ARGUMENT from `sync_status`, and books that change no more until then, if
        one of the sequences that get rows holds tokens already."""
        self._batch(sequences, offsets)
        held = self.lengths.index_select(0, sequences.clamp(0, self.lengths.shape[0] - 1))
        wrong = ((held != 0) & (offsets[1:] != offsets[:-1])).any()
        self._error.masked_fill_(wrong & (self._error == 0), _BAD_SEQUENCE)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, sequences: torch.Tensor,
               offsets: torch.Tensor) -> None:
        """Quantises the rows into their places, the last tokens of each sequence."""
        stream = self._batch(sequences, offsets)
        rows, heads, k_stride = _row_layout(k, "k", self.device)
        v_rows, v_heads, v_stride = _row_layout(v, "v", self.device)
        if v_rows != rows or heads != self.kv_heads or v_heads != heads:
            raise NmoeError(1, "KvCache.append", "k and v must be [rows, kv_heads, 128]")
        _check(_lib().nmoe_kv_append(self._ref, stream, layer, k.data_ptr(), k_stride, v.data_ptr(),
                                     v_stride, sequences.data_ptr(), offsets.data_ptr(),
                                     sequences.shape[0], rows), "nmoe_kv_append")

    def attend(self, layer: int, q: torch.Tensor, sequences: torch.Tensor, offsets: torch.Tensor,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of new rows, the last tokens of their sequences: row j of c sees every token
        up to position length - c + j.  Returns [rows, heads, 128] bf16; rows of no entry are as `out`
        had them, undefined without it."""
        stream = self._batch(sequences, offsets)
        rows, heads, q_stride = _row_layout(q, "q", self.device)
        if heads % self.kv_heads or (rows and sequences.shape[0] == 0):
            raise NmoeError(1, "KvCache.attend", "heads must be a multiple of kv_heads, rows need a sequence")
        out = _output(out, q)
        _check(_lib().nmoe_attention_cached(
            self._ref, stream, layer, q.data_ptr(), q_stride, heads, sequences.data_ptr(),
            offsets.data_ptr(), sequences.shape[0], rows, DEFAULT_SCALE if scale is None else scale,
            out.data_ptr()), "nmoe_attention_cached")
        return out

    def find_shared(self, sequences: torch.Tensor, offsets: torch.Tensor, groups: torch.Tensor,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """How many tokens the entries of a batch have in common with their groups, [n] int32, for
        `attend_shared`: entries [groups[g], groups[g + 1]) are a group, such as the children of one
        parent, and what its members with new rows share are the pages with which all their rows of the
        block table begin, before all new rows, as whole runs of 128 tokens.  0 for entries of no group,
        and where fewer than two members have rows.  Once a step, behind `extend`, for all layers."""
        stream = self._batch(sequences, offsets)
        self._groups(sequences, groups)
        if out is None:
            out = torch.empty_like(sequences)
        else:
            _require_list(out, "out", self.device)
            if out.shape != sequences.shape:
                raise ValueError("out must have as many entries as sequences")
        # (rows: the lists are within what they say themselves)
        _check(_lib().nmoe_kv_find_shared(self._ref, stream, sequences.data_ptr(), offsets.data_ptr(), sequences.shape[0],
                                          _MOST_ROWS, groups.data_ptr(), groups.shape[0] - 1, out.data_ptr()),
               "nmoe_kv_find_shared")
        return out

    def attend_shared(self, layer: int, q: torch.Tensor, sequences: torch.Tensor, offsets: torch.Tensor,
                      groups: torch.Tensor, shared: torch.Tensor, scale: Optional[float] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """`attend` for a batch in groups, with what `find_shared` found for it: the tokens that a group
        shares are read once for all of its rows.  It pays where what is not read again is some 250 MB of
        codes in a layer or more, 256 bytes a token and key head (64 continuations of 2048 tokens with 8
        key heads); below, `attend` takes less time.

        Queries are taken as two 8-bit terms, weights as two such (within 2^-8) or, for groups of
        more than 128 rows of queries to a key head, as binary16 (2^-11; 2^-25 of the largest where
        that is more); sums are FP32 and results bf16.  Each call allocates some 60 MB meanwhile."""
        stream = self._batch(sequences, offsets)
        self._groups(sequences, groups)
        _require_list(shared, "shared", self.device)
        if shared.shape != sequences.shape:
            raise ValueError("shared must have as many entries as sequences")
        rows, heads, q_stride = _row_layout(q, "q", self.device)
        if heads % self.kv_heads or (rows and sequences.shape[0] == 0):
            raise NmoeError(1, "KvCache.attend_shared", "heads must be a multiple of kv_heads, rows need a sequence")
        out = _output(out, q)
        library = _library or _lib()
        needed = library.nmoe_attention_shared_workspace_bytes(rows, heads) if rows else 0
        workspace = torch.empty(needed, dtype=torch.uint8, device=self.device)
        _check(library.nmoe_attention_shared(
            self._ref, stream, layer, q.data_ptr(), q_stride, heads, sequences.data_ptr(), offsets.data_ptr(),
            sequences.shape[0], rows, groups.data_ptr(), groups.shape[0] - 1, shared.data_ptr(),
            DEFAULT_SCALE if scale is None else scale, workspace.data_ptr(), needed, out.data_ptr()),
            "nmoe_attention_shared")
        return out

    def _groups(self, sequences: torch.Tensor, groups: torch.Tensor) -> None:
        _require_list(groups, "groups", self.device)
        if not 1 <= groups.shape[0] <= sequences.shape[0] + 1:
            raise ValueError("groups must have one entry more than there are groups, no more of them than sequences")

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """children[i] becomes a copy of parents[i]: full pages are shared, a partly filled last
        one is copied.  What a child held is given up first."""
        stream = _stream_of(self.device, "the cache")
        _require_list(parents, "parents", self.device)
        _require_list(children, "children", self.device)
        if parents.numel() != children.numel():
            raise ValueError("every child needs one parent")
        _check(_lib().nmoe_kv_fork(self._ref, stream, parents.data_ptr(), children.data_ptr(),
                                   parents.numel()), "nmoe_kv_fork")

    def free(self, sequences: torch.Tensor) -> None:
        """Gives up the sequences' pages; what nobody holds any more is free."""
        stream = _stream_of(self.device, "the cache")
        _require_list(sequences, "sequences", self.device)
        _check(_lib().nmoe_kv_free(self._ref, stream, sequences.data_ptr(), sequences.numel()),
               "nmoe_kv_free")

    def compact(self) -> None:
        """Moves the pages in use to the front of the pool, into the free ones there."""
        _check(_lib().nmoe_kv_compact(self._ref, _stream_of(self.device, "the cache")), "nmoe_kv_compact")

    def copy_pages(self, sources: torch.Tensor, targets: torch.Tensor) -> None:
        """Copies pages in every layer; no target is a source or another's target."""
        stream = _stream_of(self.device, "the cache")
        _require_list(sources, "sources", self.device)
        _require_list(targets, "targets", self.device)
        if sources.numel() != targets.numel():
            raise ValueError("every source needs one target")
        _check(_lib().nmoe_kv_copy_pages(self._ref, stream, sources.data_ptr(),
                                         targets.data_ptr(), sources.numel()), "nmoe_kv_copy_pages")

    def sync_status(self) -> int:
        """Waits for the current stream; what its calls on this cache could not do, and clears it."""
        return _lib().nmoe_kv_sync_status(self._ref, _stream())
