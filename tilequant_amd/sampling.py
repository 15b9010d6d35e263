"""Drawing tokens from logits (HIP, gfx950): temperature, top-k, top-p and min-p from given random numbers.

``sample_tokens`` stands beside the decoder's greedy step (``tq_greedy_step``; the reference decodes greedily only,
src/runtime/graph_decode.py:347-385): one call for any batch, every row with settings of its own, no host
synchronisation, so it can be captured behind a model's logits.  The rules are in ``include/tilequant.h``
(``tq_sample_tokens``), the kernel in ``csrc/tq_sample.hip``.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional, Union

import torch

from . import _native as nat

Setting = Union[float, int, torch.Tensor]

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


@lru_cache(maxsize=1024)
def _workspace_elems(rows: int, vocab: int) -> int:
    return int(nat.lib().tq_sample_workspace_elems(rows, vocab))


def _setting(name: str, value: Setting, dtype: torch.dtype, logits: torch.Tensor):
    """(pointer, value for all rows) of a setting given per row or once."""
    if isinstance(value, torch.Tensor):
        nat.require_device(value)
        if value.dtype != dtype or value.shape != logits.shape[:1] or not value.is_contiguous() \
                or value.device != logits.device:
            raise ValueError(f"{name} must be a number or a contiguous {dtype} vector with one entry per row on the "
                             "logits' device")
        return value.data_ptr(), 0
    return None, value


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Token ids [rows] (int64) drawn from ``logits`` [rows, vocab] (bf16, fp16 or fp32, any row stride; vocab up to
    500000, rows up to 65535) with one number in [0, 1) per row, ``uniform`` [rows] fp32.

    ``temperature`` (<= 0: the argmax), ``top_k`` (<= 0: all), ``top_p`` (>= 1: all) and ``min_p`` (0: all) are numbers
    or, for settings of each row's own, vectors: int32 for ``top_k``, fp32 for the others.  They apply in this
    order, top-p to the mass that top-k left, min-p to the weight beside the likeliest token's.  Tokens of equal logits
    rank by index.  The same inputs give the same ids on every call."""
    nat.require_device(logits, uniform, out)
    if logits.dim() != 2 or logits.shape[1] < 1 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows, vocab] with unit column stride")
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {logits.dtype}; expected bfloat16, float16 or float32")
    rows, vocab = logits.shape
    if rows > 1 and logits.stride(0) < vocab:
        raise ValueError("rows of logits overlap")
    if uniform.dtype != torch.float32 or uniform.shape != (rows,) or not uniform.is_contiguous() \
            or uniform.device != logits.device:
        raise ValueError("uniform must be a contiguous fp32 vector with one entry per row on the logits' device")
    t, t_all = _setting("temperature", temperature, torch.float32, logits)
    k, k_all = _setting("top_k", top_k, torch.int32, logits)
    p, p_all = _setting("top_p", top_p, torch.float32, logits)
    m, m_all = _setting("min_p", min_p, torch.float32, logits)
    if out is None:
        out = torch.empty((rows,), dtype=torch.int64, device=logits.device)
    elif out.dtype != torch.int64 or out.shape != (rows,) or not out.is_contiguous() or out.device != logits.device:
        raise ValueError("out must be a contiguous int64 vector with one entry per row on the logits' device")
    # scratch of this call alone: calls on other streams, and graphs, have their own
    elems = _workspace_elems(rows, vocab)
    workspace = torch.empty((elems,), dtype=torch.int64, device=logits.device) if elems else None
    nat.launch(logits.device, "tq_sample_tokens", nat.lib().tq_sample_tokens,
               logits.data_ptr(), logits.stride(0), code, rows, vocab, uniform.data_ptr(), t, float(t_all), k, min(max(int(k_all), 0), vocab),
               p, float(p_all), m, float(m_all), out.data_ptr(), nat.ptr(workspace), elems)
    return out
