"""Choice of a token per row of logits with temperature, top-k, top-p and min-p from given random numbers, on the device.

The reference takes the recogniser's tokens from its pipeline call (/root/reference/voice-service/app/services/
voice_interface.py:2049-2053), whose choice is the arg-max (``ParaformerHead``); ``sample_tokens`` stands beside it for models
that draw.  The random numbers are an input, so a call's result is a function of its arguments.
"""
from __future__ import annotations

import torch

from . import _lib

_DT = {torch.float32: _lib.DT_F32, torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}
MAX_VOCAB = 1 << 18


def _per_row(name, value, rows, dtype, index, device):
    """A setting for every row: a tensor [rows], one number for all, or None."""
    if value is None:
        return None
    if not isinstance(value, torch.Tensor):
        return torch.full((rows,), value, dtype=dtype, device=device)
    if value.dtype is not dtype or value.dim() != 1 or value.shape[0] != rows or value.get_device() != index or not value.is_contiguous():
        raise ValueError(f"sample_tokens: {name} must be one number or a contiguous {dtype} tensor [{rows}] on {device}")
    return value


def _ptr(t):
    return None if t is None else t.data_ptr()


def sample_tokens(ctx: _lib.Context, logits: torch.Tensor, u: torch.Tensor, temperature=None, top_k=None, top_p=None, min_p=None,
                  token_num: torch.Tensor | None = None, ids: torch.Tensor | None = None):
    """logits [rows, vocab] (float32, float16 or bfloat16, rows of contiguous elements at any stride) and u [rows] float32 in
    [0, 1) -> (ids [rows] int32, logprobs [rows] float32).

    Weights are exp((l - max l) / temperature).  In the order of falling logits (equal ones by rising index) the first ``top_k``
    are kept (<= 0: all), of those the shortest prefix with at least ``top_p`` of their weight, of those the ones with at
    least ``min_p`` of the largest weight, and always the first; the id is the lowest one at which the running sum of the
    kept weights exceeds ``u`` times their sum.  A temperature that is not above zero takes the arg-max, one
    above 1e30 counts as 1e30.  Every setting is one number (u, too), a tensor [rows] or None.  NaN logits count as -inf; a row with nothing above -inf gives id 0 and logprob -inf.
    ``token_num`` [rows / n] int32: of every n rows the ones behind an utterance's tokens get id -1 and logprob 0."""
    if not logits.is_cuda or logits.dtype not in _DT or logits.dim() != 2 or not 1 <= logits.shape[1] <= MAX_VOCAB:
        raise ValueError(f"sample_tokens: logits must be a float32, float16 or bfloat16 CUDA tensor [rows, 1 .. {MAX_VOCAB}]")
    rows, vocab = logits.shape
    stride, step = logits.stride()
    index, dev = logits.get_device(), logits.device
    if rows and vocab > 1 and step != 1 or rows > 1 and stride < vocab:
        raise ValueError("sample_tokens: every row's logits must lie side by side, rows must not overlap")
    u = _per_row("u", u, rows, torch.float32, index, dev)
    temperature = _per_row("temperature", temperature, rows, torch.float32, index, dev)
    top_k = _per_row("top_k", top_k, rows, torch.int32, index, dev)
    top_p = _per_row("top_p", top_p, rows, torch.float32, index, dev)
    min_p = _per_row("min_p", min_p, rows, torch.float32, index, dev)
    if u is None:
        raise ValueError("sample_tokens: u is needed")
    rows_per = 0
    if token_num is not None:
        if token_num.dtype != torch.int32 or token_num.dim() != 1 or token_num.get_device() != index or not token_num.is_contiguous() \
                or not token_num.shape[0] or rows % token_num.shape[0] or not rows:
            raise ValueError("sample_tokens: token_num must be a contiguous int32 tensor whose length divides the rows")
        rows_per = rows // token_num.shape[0]
    if ids is None:
        ids = torch.empty((rows,), dtype=torch.int32, device=dev)
    elif ids.dtype != torch.int32 or ids.shape != (rows,) or ids.get_device() != index or not ids.is_contiguous():
        raise ValueError(f"sample_tokens: ids must be a contiguous int32 tensor [{rows}] on {dev}")
    logprobs = torch.empty((rows,), dtype=torch.float32, device=dev)
    if rows:
        if torch.cuda.current_device() != index:
            with torch.cuda.device(index):
                return sample_tokens(ctx, logits, u, temperature, top_k, top_p, min_p, token_num, ids)
        rc = ctx.lib.asrfe_sample_tokens(
            ctx.handle, logits.data_ptr(), _DT[logits.dtype], stride if rows > 1 else vocab, rows, vocab, u.data_ptr(), _ptr(temperature),
            _ptr(top_k), _ptr(top_p), _ptr(min_p), _ptr(token_num), rows_per, ids.data_ptr(), logprobs.data_ptr(), _lib.raw_stream(index))
        if rc:
            ctx.check(rc)
    return ids, logprobs
