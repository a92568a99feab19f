"""Causal attention over whole prompts (the prefill or extend step) of packed sequences.

The reference accelerates the decode only; its adapter inherits SGLang's extend step
(``integrations/sglang_backend.py:14-108``).  ``prompt_attention`` is that step for the same
caches: packed keys of fresh prompts, or cache slots when part of a sequence is cached already.
"""
from __future__ import annotations

import torch

from . import _native


def prompt_attention(q, k, v, indptr, *, kv_indptr=None, kv_indices=None, scale=None, logit_cap=0.0, window_left=-1,
                     out=None, lse=None, status=None):
    """Each query of ``q`` [T, Hq, D] attends to its own sequence up to its own position.

    Sequence i owns query rows ``indptr[i]`` to ``indptr[i + 1]`` (int32, on the GPU; the host never
    reads it) and the keys ``kv_indptr[i]`` to ``kv_indptr[i + 1]`` (``indptr`` where absent); its last
    query sits at its last key, so earlier keys are a cached past.  Key number x is row x of
    ``k`` / ``v`` [N, Hkv, D], or row ``kv_indices[x]`` (int32) of a cache with one-token pages, as in
    ``DecodeEngine.execute``; a row outside ``k`` reads as zeros.  fp16 or bf16, D 64, 128 or 256,
    1 to 16 query heads per KV head, any strides (rows 16-byte aligned with unit stride along D
    run on the tcgen05 kernel for D 64 and 128, others on a slower one).

    ``scale`` (> 0) defaults to D^-0.5; ``logit_cap`` > 0 soft-caps scores, s -> cap * tanh(s / cap);
    ``window_left`` >= 0 lets a query see its last window_left + 1 keys only.  A query without
    any key (a sequence with fewer keys than queries) gives zeros.  A value that is not finite
    reaches the rows that see it and no others.  Rows of ``out`` (allocated when absent; it must not
    share memory with the inputs) outside the sequences are left as they were.  ``lse`` (fp32 [T, Hq], optional) receives
    each row's natural-log sum of exponentials, -inf without a key; ``status`` (int32[1], optional)
    is set non-zero if an in-kernel wait expires (4 s; every row that this kept from being computed is then
    NaN, and some of the same thread block's others).

    Scores, softmax and sums are fp32; the weights are rounded to q's dtype for their product with
    ``v``.  Returns ``out``.
    """
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _native.op("prompt_attention")(q, k, v, indptr, kv_indptr, kv_indices, out, lse,
                                   q.shape[-1] ** -0.5 if scale is None else float(scale), float(logit_cap or 0.0),
                                   int(window_left), status)
    return out
