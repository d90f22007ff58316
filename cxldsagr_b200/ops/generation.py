"""Operators of drawing several continuations of one committed history.

:func:`shared_prefix_mla` attends a batch of continuations to the history rows
they share (read once for all of them) and to each one's own tail;
:func:`sample_tokens` draws one token per row of logits.  CUDA tensors run the
native kernels, CPU tensors the oracles of :mod:`.reference`.
"""

from __future__ import annotations

import math

import torch

from . import reference
from .native import lib


def _records_ok(t: torch.Tensor) -> bool:
    """Rows the kernels can load: contiguous records that start on 16-byte boundaries."""
    if t.data_ptr() % 16:
        return False
    if t.numel() == 0:
        return True
    return t.stride(-1) == 1 and all(n == 1 or (s >= 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride()))


def shared_prefix_mla(q, prefix, tail, tail_lens, scale, *, return_lse: bool = False, value_dim: int = 512):
    """MLA of B continuations over one shared prefix and their own tails.

    ``q``          [B, H, 576] (one new token each) or [B, T, H, 576] absorbed queries, BF16;
    ``prefix``     [P, 576] records every continuation sees (P may be 0; rows may be strided);
    ``tail``       [B, S, 576] own records (strided views are fine) or None;
    ``tail_lens``  int32 [B], the tail rows visible to the last query token of
                   each continuation (0 <= len <= S), or None for all S.  Query
                   token t sees ``len - (T - 1 - t)`` of them (causal inside the
                   tail).  Rows past the visible ones are never used, whatever they hold.

    Returns BF16 [..., H, 512]: softmax over the visible records of
    ``scale * q . k``, times the records' first ``value_dim`` dims.  A query that
    sees no record gives zeros.  With ``return_lse`` also the FP32 natural-log
    sum of exponentials [..., H] (-inf where nothing is visible), to merge with
    other parts of the attention.  On CUDA a length outside [0, S] is recorded
    in the device error word (``check_errors``) and clamped.
    """
    if q.dim() not in (3, 4):
        raise ValueError("q must be [B, H, D] or [B, T, H, D]")
    B, D = q.shape[0], q.shape[-1]
    if prefix.dim() != 2 or prefix.shape[1] != D:
        raise ValueError("prefix must be [P, D] with the query's record width")
    if tail is None:
        if tail_lens is not None:
            raise ValueError("tail_lens needs a tail")
    elif tail.dim() != 3 or tail.shape[0] != B or tail.shape[2] != D:
        raise ValueError("tail must be [B, S, D] with the query's batch and record width")
    if tail_lens is not None and (tail_lens.dim() != 1 or tail_lens.shape[0] != B):
        raise ValueError("tail_lens must be [B]")
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError("scale must be positive and finite")
    tensors = [t for t in (q, prefix, tail, tail_lens) if t is not None]
    if any(t.device != q.device for t in tensors):
        raise ValueError("q, prefix, tail and tail_lens must be on one device")
    if not q.is_cuda:
        out, lse = reference.shared_prefix_mla(q, prefix, tail, tail_lens, scale, value_dim)
        return (out, lse) if return_lse else out
    if value_dim != 512 or D != 576:
        raise ValueError("the sm_100a shared-prefix MLA kernel covers the V3.2 shape (576 / 512)")
    if any(t.dtype != torch.bfloat16 for t in (q, prefix) + (() if tail is None else (tail,))):
        raise ValueError("q, prefix and tail must be BF16")
    for name, t in (("prefix", prefix), ("tail", tail)):
        if t is not None and not _records_ok(t):
            raise ValueError(f"{name} records must be contiguous and start on 16-byte boundaries")
    if tail_lens is not None and tail_lens.dtype != torch.int32:
        raise ValueError("tail_lens must be int32")
    q4 = (q if q.dim() == 4 else q.unsqueeze(1)).contiguous()
    out = torch.empty((*q4.shape[:3], 512), dtype=torch.bfloat16, device=q.device)
    lse = torch.empty(q4.shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
    lib().shared_prefix_mla(q4, prefix, tail, None if tail_lens is None else tail_lens.contiguous(), float(scale), out,
                            lse)
    out = out.view(*q.shape[:-1], 512)
    return (out, lse.view(q.shape[:-1])) if return_lse else out


def _sample_param(name, value, R, dtype, device, ok):
    """(per-row tensor or None, scalar) of a sampling parameter; scalars are checked, device values are not."""
    if torch.is_tensor(value):
        if value.dim() != 1 or value.shape[0] != R or value.device != device:
            raise ValueError(f"{name} must be a number or an [R] tensor on the logits' device")
        if value.dtype != dtype:
            raise ValueError(f"a per-row {name} must be {dtype}")
        return value.contiguous(), 0
    if not ok(value):
        raise ValueError(f"{name} out of range: {value!r}")
    return None, value


def sample_tokens(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Draw one token per row of ``logits`` [R, V] (FP32 or BF16) from the uniform numbers ``u`` [R] in [0, 1).

    With x the logits (NaN counts as -inf), d = (x - max x) / temperature, w =
    exp(d) and masses floor(2^36 w), the kept tokens are those prefixes of the
    order (x descending, then index ascending) that all filters allow: the
    first ``top_k`` (0: all); those whose preceding mass is below ``top_p``
    times the mass left by top-k (1: all); those with w >= ``min_p`` (relative
    to the best token; 0: all).  The best token is always kept.  The result is
    the first token, in vocabulary order, whose cumulative kept mass exceeds
    floor(u * total).  The masses are whole numbers, so a draw depends neither
    on the batch it is part of nor on how the sums are split.

    ``temperature`` 0 takes the best token (the first of equal ones).  Each
    parameter is a number or an [R] tensor on the logits' device (FP32; int32
    for ``top_k``); numbers are checked here, tensors are not: there a
    temperature that is not positive counts as 0, a ``top_k`` below 1 and a
    ``top_p`` or ``min_p`` that is NaN switch that filter off.

    Returns (tokens int64 [R], log-probabilities FP32 [R] of the drawn tokens
    under the filtered distribution; 0 for temperature 0).  A row whose logits
    are all -inf or NaN gives token -1 with log-probability -inf.
    """
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError("logits must be [R, V] with V >= 1")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("logits must be FP32 or BF16")
    R = logits.shape[0]
    dev = logits.device
    if u.dim() != 1 or u.shape[0] != R or u.device != dev or u.dtype != torch.float32:
        raise ValueError("u must be an FP32 [R] tensor on the logits' device")
    t_t, t_0 = _sample_param("temperature", temperature, R, torch.float32, dev, lambda v: 0 <= v < math.inf)
    k_t, k_0 = _sample_param("top_k", top_k, R, torch.int32, dev, lambda v: isinstance(v, int) and v >= 0)
    p_t, p_0 = _sample_param("top_p", top_p, R, torch.float32, dev, lambda v: 0 <= v <= 1)
    m_t, m_0 = _sample_param("min_p", min_p, R, torch.float32, dev, lambda v: 0 <= v <= 1)
    if not logits.is_cuda:
        return reference.sample_tokens(logits, u, t_0 if t_t is None else t_t, k_0 if k_t is None else k_t,
                                       p_0 if p_t is None else p_t, m_0 if m_t is None else m_t)
    if logits.shape[1] > lib().sample_max_vocabulary():
        raise ValueError(f"the sampling kernel takes vocabularies of up to {lib().sample_max_vocabulary()}")
    if logits.stride(1) != 1 and logits.shape[1] > 1:
        logits = logits.contiguous()
    tokens = torch.empty(R, dtype=torch.int64, device=dev)
    logprobs = torch.empty(R, dtype=torch.float32, device=dev)
    lib().sample_tokens(logits, u.contiguous(), t_t, k_t, p_t, m_t, float(t_0), min(int(k_0), 2**31 - 1), float(p_0),
                        float(m_0), tokens, logprobs)
    return tokens, logprobs
