"""Tokens from logits, behind the last layer of a step (`nmoe_sample`, include/nmoe.h).

    tokens = sample(logits, uniform, temperature=0.7, top_p=0.95)
    tokens, logprobs = sample(logits, uniform, temperature=temperatures, top_k=top_ks,
                              return_logprobs=True)     # a request's own parameters

`uniform` are the caller's random numbers, so a step can be repeated or recorded in a CUDA graph
(which reads what the tensors hold when it is replayed).  Calls run on the current stream and keep
nothing between them.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import NMOE_BF16, NMOE_F32, _check, load_library
from .attention import _stream_of

Parameter = Optional[Union[float, torch.Tensor]]

_library = None


def _lib() -> ctypes.CDLL:
    global _library
    if _library is None:
        lib = load_library()
        vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
        lib.nmoe_sample.argtypes = [vp, vp, ctypes.c_int, i64, i64, i32, vp, vp, f32, vp, i32, vp, f32, vp,
                                    f32, vp, vp]
        _library = lib
    return _library


def _vector(t: torch.Tensor, name: str, dtype: torch.dtype, rows: int, device: torch.device) -> int:
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != rows or t.device != device or \
            not (t.is_contiguous() or rows < 2):
        raise ValueError(f"{name} must be a contiguous vector of {rows} {dtype} on {device}")
    return t.data_ptr()


def _parameter(value: Parameter, name: str, dtype: torch.dtype, default, rows: int, device: torch.device):
    """The address of the rows' values, and one for all of them."""
    if value is None:
        return None, default
    if isinstance(value, torch.Tensor):
        return _vector(value, name, dtype, rows, device), default
    if value != value:
        raise ValueError(f"{name} is not a number")
    return None, value


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature: Parameter = None, top_k: Parameter = None,
           top_p: Parameter = None, min_p: Parameter = None, return_logprobs: bool = False,
           out: Optional[torch.Tensor] = None):
    """A token [rows] (int32) for each row of `logits` [rows, vocab], FP32 or bf16; rows may lie further
    apart than they are long.  `uniform` [rows] FP32, in [0, 1).

    The tokens are put in falling order of their logits, equal ones by rising number.  Of these the
    first `top_k` stay (all: None or below 1); of these as many as reach `top_p` of the sum of their
    weights exp(logit / temperature) (all: None or 1); of these those of at least `min_p` times the
    largest weight.  What is left shares out [0, 1) in rising order of the tokens, and `uniform`
    falls on one.  A temperature of 0 takes the first of the largest logits.  Each parameter is a
    number for all rows or a tensor with one for each (FP32, top_k int32).

    With `return_logprobs` also the FP32 logarithm [rows] of the token's probability under softmax of
    all logits, at temperature 1.  Rows with a NaN, or whose largest logit is infinite (a mask that
    leaves nothing), get token -1 and NaN."""
    device = logits.device
    stream = _stream_of(device, "logits")
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, vocab], float32 or bfloat16")
    rows, vocab = logits.shape
    if rows and (logits.stride(1) != 1 and vocab > 1 or rows > 1 and logits.stride(0) < vocab):
        raise ValueError("the logits of a row must lie side by side, rows one behind the other")
    at_uniform = _vector(uniform, "uniform", torch.float32, rows, device)
    at_temperature, temperature = _parameter(temperature, "temperature", torch.float32, 1.0, rows, device)
    at_top_k, top_k = _parameter(top_k, "top_k", torch.int32, 0, rows, device)
    at_top_p, top_p = _parameter(top_p, "top_p", torch.float32, 1.0, rows, device)
    at_min_p, min_p = _parameter(min_p, "min_p", torch.float32, 0.0, rows, device)
    if not -2 ** 31 <= top_k < 2 ** 31 or top_k != int(top_k):
        raise ValueError("top_k must be a whole number")
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=device)
    else:
        _vector(out, "out", torch.int32, rows, device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=device) if return_logprobs else None
    _check((_library or _lib()).nmoe_sample(
        stream, logits.data_ptr(), NMOE_BF16 if logits.dtype is torch.bfloat16 else NMOE_F32,
        logits.stride(0) if rows > 1 else vocab, rows, vocab, at_uniform, at_temperature, temperature, at_top_k,
        int(top_k), at_top_p, top_p, at_min_p, min_p, out.data_ptr(),
        None if logprobs is None else logprobs.data_ptr()), "nmoe_sample")
    return (out, logprobs) if return_logprobs else out
