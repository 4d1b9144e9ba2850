"""Sampling a token for each row of logits (csrc/ops/sample.hip): the sampled sibling of ``decode_tail``'s argmax."""

from __future__ import annotations

import torch

from k8s_vgpu_scheduler_amd import ops
from k8s_vgpu_scheduler_amd.ops.paged import _BF16, _F32, _I32, _I64, _launch, _ptrs

MAX_VOCAB = 128 * 32768      # csrc/ops/sample.hip CARRIES * CARRY


def sample_workspace(rows: int, vocab: int, device="cuda") -> torch.Tensor:
    """Workspace of ``sample`` for up to ``rows`` rows of ``vocab`` logits.  Empty: a row is counted and searched within
    one workgroup."""
    if rows < 1 or not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"sample_workspace: {rows} rows of {vocab} logits (at most {MAX_VOCAB})")
    return torch.empty(0, dtype=_I64, device=device)


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature: torch.Tensor | None = None,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
           tokens: torch.Tensor | None = None, probs: torch.Tensor | None = None, work: torch.Tensor | None = None):
    """One token a row -> (tokens int64 [B], probs fp32 [B]: its probability among the kept).

    logits bf16 [B, V] (unit column stride), uniform fp32 [B] in [0, 1), and for each row, or None for off:
    temperature fp32 (1; at or below 0: the first maximum), top_k int32 (at or below 0: off), top_p fp32 (from 1:
    off), min_p fp32.  In the order of larger logits (equal ones: lower index), with weights exp((l - max) / T):
    the first top_k, of these the smallest prefix that has top_p of their weight, of these the ones of at least min_p
    times the largest weight (the first stays in any case, alone where min_p is above 1); the answer is the first whose
    running sum of weights exceeds uniform times their sum.
    -inf is a masked token; a row of nothing else gives -1 (probability 0).  A NaN counts as the maximum, as in
    ``decode_tail`` (probability NaN).  ``work`` from ``sample_workspace``."""
    if logits.dim() != 2:
        raise ValueError(f"sample: logits must be [B, V], got {tuple(logits.shape)}")
    B, V = logits.shape
    if logits.dtype is not _BF16 or B < 1 or not 0 < V <= MAX_VOCAB or (V > 1 and logits.stride(1) != 1) \
            or (B > 1 and logits.stride(0) < V):
        raise ValueError(f"sample: logits must be bf16 [B, V <= {MAX_VOCAB}] with unit column stride, got "
                         f"{logits.dtype} {list(logits.shape)} strides {list(logits.stride())}")
    if tokens is None:
        tokens = torch.empty(B, dtype=_I64, device=logits.device)
    if probs is None:
        probs = torch.empty(B, dtype=_F32, device=logits.device)
    idx, p = _ptrs("sample", ("uniform", uniform, _F32, (B,)), ("temperature", temperature, _F32, (B,)),
                   ("top_k", top_k, _I32, (B,)), ("top_p", top_p, _F32, (B,)), ("min_p", min_p, _F32, (B,)),
                   ("tokens", tokens, _I64, (B,)), ("probs", probs, _F32, (B,)))
    if logits.get_device() != idx:
        raise ValueError(f"sample: logits are on {logits.device}: every tensor must be on one GPU")
    if work is not None and (work.dtype is not _I64 or work.get_device() != idx):
        raise ValueError(f"sample: work must be from sample_workspace on {logits.device}")
    _launch(idx, "sample", ops.lib().mivgpu_sample, logits.data_ptr(), logits.stride(0) if B > 1 else V, V, B, *p)
    return tokens, probs
