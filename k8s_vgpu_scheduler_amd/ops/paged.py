"""Batched serving on a paged 8-bit K/V cache (csrc/ops/paged_*.hip).

A serving step over a batch of requests of different lengths:

    plan = pool.plan(new_lens, n_tokens)                 # pages, slots, positions: once for all layers
    for each layer:
        ops.paged_qk_norm_rope_kv(qkv, ..., plan.positions, plan.slots, turns, cache, q, ...)
        ops.paged_attention(q, cache, pool.table, plan.cu_q, plan.kv_lens, ...)
    tokens, probs = ops.sample(logits, uniform, temperature, top_k, top_p, min_p)
    pool.commit(plan, finished)                          # the step is done: lengths and pages move on

The step's tokens are packed: request b owns rows ``cu_q[b] .. cu_q[b+1]``; rows behind the last request are left
as they are.  K and V are e4m3 codes with one power-of-two scale for each page of 64 tokens and kv head.
Everything is static in shape and runs on the caller's stream without a host synchronisation, so a step can be
captured by ``torch.cuda.CUDAGraph``.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from k8s_vgpu_scheduler_amd import ops

PAGE = 64            # tokens of a page (csrc/ops/paged.h)
MAX_ROWS = 1024      # requests of one call


def _on(device: torch.device, name: str, **tensors):
    """Every tensor on ``device``, of its type, contiguous: ``name=(tensor, dtype)``."""
    if device.type != "cuda":
        raise ValueError(f"{name}: tensors must be on the GPU, got {device}")
    for what, (t, dtype) in tensors.items():
        if t is None:
            continue
        if t.device != device or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{name}: {what} must be contiguous {dtype} on {device}, got "
                             f"{tuple(t.shape)} {t.dtype} on {t.device}")


def _launch(device, name, fn, *args):
    """The C call on ``device``'s current stream, whatever the current device is."""
    with torch.cuda.device(device):
        ops._check(fn(*args, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), name)


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


# ------------------------------------------------------------------ pages --
class PagePlan(NamedTuple):
    """What a step needs to know about its tokens (all int32, on the GPU).

    cu_q [B+1]        row of each request's first token (prefix sums of the new lengths)
    kv_lens [B]       keys of each request after the step; 0 where it is not admitted
    taken [B]         new pages of each request; -1 where it is not admitted
    positions [N]     position of each token; 0 for rows without a request
    slots [N]         page * 64 + place of each token; -1 for rows without a request or of one not admitted
    """
    cu_q: torch.Tensor
    kv_lens: torch.Tensor
    taken: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


def page_plan(new_lens: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, free: torch.Tensor,
              ring: torch.Tensor, n_tokens: int, out: PagePlan | None = None) -> PagePlan:
    """Pages for ``new_lens[b]`` new tokens of requests that hold ``lengths[b]`` (int32 [B], B <= 1024; a negative
    one counts as 0).

    table int32 [B, W]: pages of each request; the new ones are written behind the committed ones.  free int32
    [pages], ring int32 [2]: the free pages are ``free[(ring[0] + i) % pages]``, i < ring[1].  A request is admitted
    if its tokens fit (64 * W of them, and ``n_tokens`` rows in all) and the free pages reach for the pages of every
    request up to it; what it would have taken stays reserved for it ahead of later ones.  Nothing that is committed
    changes: planning again gives the same plan, and ``page_commit`` makes it so."""
    B = new_lens.numel()
    dev = new_lens.device
    i32 = torch.int32
    _on(dev, "page_plan", new_lens=(new_lens, i32), lengths=(lengths, i32), table=(table, i32), free=(free, i32),
        ring=(ring, i32))
    if not 0 < B <= MAX_ROWS or new_lens.dim() != 1 or tuple(lengths.shape) != (B,) or table.dim() != 2 \
            or table.shape[0] != B or table.shape[1] < 1 or free.dim() != 1 or free.numel() < 1 or tuple(ring.shape) != (2,):
        raise ValueError(f"page_plan: new_lens / lengths [B <= {MAX_ROWS}], table [B, W], free [pages], ring [2]; got "
                         f"{tuple(new_lens.shape)} {tuple(lengths.shape)} {tuple(table.shape)} {tuple(free.shape)} "
                         f"{tuple(ring.shape)}")
    if n_tokens < 0 or max(free.numel(), table.shape[1]) * PAGE > 2**31 - 1:
        raise ValueError(f"page_plan: n_tokens {n_tokens}, {free.numel()} pages, {table.shape[1]} a request: slots are "
                         "32-bit")
    if out is None:
        buf = torch.empty(3 * B + 1 + 2 * n_tokens, dtype=i32, device=dev)     # one allocation
        out = PagePlan(*buf.split([B + 1, B, B, n_tokens, n_tokens]))
    else:
        _on(dev, "page_plan", **{n: (t, i32) for n, t in zip(PagePlan._fields, out)})
        if [t.numel() for t in out] != [B + 1, B, B, n_tokens, n_tokens]:
            raise ValueError(f"page_plan: out must hold {B + 1}, {B}, {B}, {n_tokens}, {n_tokens} values")
    _launch(dev, "page_plan", ops.lib().mivgpu_page_plan, _ptr(new_lens), _ptr(lengths), _ptr(table), _ptr(free),
            _ptr(ring), *map(_ptr, out), B, table.shape[1], free.numel(), n_tokens)
    return out


def page_commit(plan: PagePlan, lengths: torch.Tensor, table: torch.Tensor, free: torch.Tensor, ring: torch.Tensor,
                finished: torch.Tensor | None = None):
    """The plan's step is done: ``lengths`` of admitted requests become its ``kv_lens`` and their pages leave the
    ring.  ``finished`` (bool [B]): requests whose pages go back to the ring's end, in order; their length becomes 0."""
    B = lengths.numel()
    dev = lengths.device
    i32 = torch.int32
    _on(dev, "page_commit", lengths=(lengths, i32), table=(table, i32), free=(free, i32), ring=(ring, i32),
        kv_lens=(plan.kv_lens, i32), taken=(plan.taken, i32), finished=(finished, torch.bool))
    if not 0 < B <= MAX_ROWS or lengths.dim() != 1 or tuple(plan.kv_lens.shape) != (B,) or tuple(plan.taken.shape) != (B,) \
            or table.dim() != 2 or table.shape[0] != B or free.dim() != 1 or free.numel() < 1 \
            or tuple(ring.shape) != (2,) or (finished is not None and tuple(finished.shape) != (B,)):
        raise ValueError(f"page_commit: a plan, table and finished of {B} requests, free [pages], ring [2]")
    _launch(dev, "page_commit", ops.lib().mivgpu_page_commit, _ptr(plan.kv_lens), _ptr(plan.taken), _ptr(finished),
            _ptr(lengths), _ptr(table), _ptr(free), _ptr(ring), B, table.shape[1], free.numel())


class PagePool:
    """The pages of a server: ``rows`` requests at once, each of at most ``max_pages`` pages, out of ``num_pages``
    that all layers' caches share."""

    def __init__(self, num_pages: int, rows: int, max_pages: int, device="cuda"):
        if num_pages < 1 or not 0 < rows <= MAX_ROWS or max_pages < 1:
            raise ValueError(f"PagePool: {num_pages} pages, {rows} rows (at most {MAX_ROWS}), {max_pages} pages a row")
        i32 = dict(dtype=torch.int32, device=device)
        self.lengths = torch.zeros(rows, **i32)
        self.table = torch.full((rows, max_pages), -1, **i32)
        self.free = torch.arange(num_pages, **i32)
        self.ring = torch.tensor([0, num_pages], **i32)

    def plan(self, new_lens: torch.Tensor, n_tokens: int, out: PagePlan | None = None) -> PagePlan:
        return page_plan(new_lens, self.lengths, self.table, self.free, self.ring, n_tokens, out)

    def commit(self, plan: PagePlan, finished: torch.Tensor | None = None):
        page_commit(plan, self.lengths, self.table, self.free, self.ring, finished)


class PagedKV(NamedTuple):
    """One layer's K and V: codes k [pages, Hkv, 64, D], v [pages, Hkv, D, 64] (torch.float8_e4m3fn), scales
    k_scale, v_scale [pages, Hkv] fp32 (powers of two); a value is its code times its page's scale."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def paged_kv_cache(num_pages: int, n_kv_heads: int, head_dim: int, device="cuda") -> PagedKV:
    """An empty cache (unwritten slots are never read)."""
    if num_pages < 1 or n_kv_heads < 1 or head_dim not in (64, 128):
        raise ValueError(f"paged_kv_cache: {num_pages} pages, {n_kv_heads} heads of {head_dim} (64 or 128)")
    code = dict(dtype=torch.float8_e4m3fn, device=device)
    scale = dict(dtype=torch.float32, device=device)
    return PagedKV(torch.empty(num_pages, n_kv_heads, PAGE, head_dim, **code),
                   torch.empty(num_pages, n_kv_heads, head_dim, PAGE, **code),
                   torch.empty(num_pages, n_kv_heads, **scale), torch.empty(num_pages, n_kv_heads, **scale))


def _check_cache(cache: PagedKV, device, name, n_q_heads, n_kv_heads, head_dim) -> int:
    """Host check of the cache's layout and the head counts; returns its pages."""
    if n_kv_heads < 1 or n_q_heads < 1 or n_q_heads % n_kv_heads or head_dim not in (64, 128):
        raise ValueError(f"{name}: {n_q_heads} / {n_kv_heads} heads of {head_dim} (64 or 128)")
    _on(device, name, k=(cache.k, torch.float8_e4m3fn), v=(cache.v, torch.float8_e4m3fn),
        k_scale=(cache.k_scale, torch.float32), v_scale=(cache.v_scale, torch.float32))
    pages = cache.k.shape[0]
    if tuple(cache.k.shape) != (pages, n_kv_heads, PAGE, head_dim) or tuple(cache.v.shape) != (pages, n_kv_heads, head_dim, PAGE) \
            or tuple(cache.k_scale.shape) != (pages, n_kv_heads) or tuple(cache.v_scale.shape) != (pages, n_kv_heads):
        raise ValueError(f"{name}: cache k {tuple(cache.k.shape)}, v {tuple(cache.v.shape)}, scales "
                         f"{tuple(cache.k_scale.shape)} {tuple(cache.v_scale.shape)} do not match {n_kv_heads} heads of "
                         f"{head_dim}")
    if pages < 1 or pages * PAGE > 2**31 - 1:
        raise ValueError(f"{name}: {pages} pages: slots are 32-bit")
    return pages


# ----------------------------------------------------------------- append --
def rope_turns(theta: float, head_dim: int, device="cuda") -> torch.Tensor:
    """The rotation's table: 2^64 * theta^(-2i/D) / 2pi for i < D/2, rounded, modulo 2^64 (int64 bits).  A
    position's angle in turns is the fraction position * turns / 2^64, exact to 2^-65 of the position."""
    if head_dim not in (64, 128) or not theta > 0:
        raise ValueError(f"rope_turns: theta {theta}, head_dim {head_dim} (64 or 128)")
    vals = [round(theta ** (-2.0 * i / head_dim) / (2 * math.pi) * 2**64) % 2**64 for i in range(head_dim // 2)]
    return torch.tensor([v - 2**64 if v >= 2**63 else v for v in vals], dtype=torch.int64, device=device)


def paged_qk_norm_rope_kv(qkv: torch.Tensor, q_norm_w: torch.Tensor, k_norm_w: torch.Tensor, positions: torch.Tensor,
                          slots: torch.Tensor, turns: torch.Tensor, cache: PagedKV, q_out: torch.Tensor, n_q_heads: int,
                          n_kv_heads: int, head_dim: int, eps: float):
    """Packed tokens qkv [N, (Hq+2Hkv)*D] bf16 (rows may be strided, by a multiple of 8) -> per-head RMSNorm of q and
    k, NeoX RoPE at ``positions`` [N] -> q_out [N, Hq, D] bf16; K and V appended to ``cache`` at ``slots`` [N].

    A row whose slot is outside the cache appends nothing (its q_out is written).  Tokens of one page stand together,
    in the order of their slots, behind the page's live tokens: a page whose first slot is written starts afresh, any
    other keeps its earlier tokens, whose codes follow when a new value raises the page's scale.  (``PagePool.plan``
    gives such slots.)  A token whose K or V of a head is not finite is stored as NaN in K and zero in V."""
    N = positions.numel()
    dev = qkv.device
    pages = _check_cache(cache, dev, "paged_qk_norm_rope_kv", n_q_heads, n_kv_heads, head_dim)
    bf = torch.bfloat16
    width = (n_q_heads + 2 * n_kv_heads) * head_dim
    _on(dev, "paged_qk_norm_rope_kv", q_norm_w=(q_norm_w, bf), k_norm_w=(k_norm_w, bf), positions=(positions, torch.int32),
        slots=(slots, torch.int32), turns=(turns, torch.int64), q_out=(q_out, bf))
    if qkv.dtype != bf or qkv.dim() != 2 or tuple(qkv.shape) != (N, width) or (N > 0 and qkv.stride(1) != 1) \
            or (N > 1 and (qkv.stride(0) % 8 or qkv.stride(0) < width)):
        raise ValueError(f"paged_qk_norm_rope_kv: qkv must be bf16 [{N}, {width}] with unit column stride and a row stride "
                         f"that is a multiple of 8, got {tuple(qkv.shape)} {qkv.dtype} strides {qkv.stride()}")
    if tuple(positions.shape) != (N,) or tuple(slots.shape) != (N,) or q_norm_w.numel() != head_dim \
            or k_norm_w.numel() != head_dim or turns.numel() != head_dim // 2 \
            or tuple(q_out.shape) != (N, n_q_heads, head_dim):
        raise ValueError(f"paged_qk_norm_rope_kv: positions / slots [{N}], norm weights [{head_dim}], turns "
                         f"[{head_dim // 2}], q_out [{N}, {n_q_heads}, {head_dim}]")
    for what, t in (("qkv", qkv), ("q_norm_w", q_norm_w), ("k_norm_w", k_norm_w), ("q_out", q_out), ("k", cache.k),
                    ("v", cache.v)):
        if N > 0 and t.data_ptr() % 16:
            raise ValueError(f"paged_qk_norm_rope_kv: {what} must start at a multiple of 16 bytes")
    _launch(dev, "paged_qk_norm_rope_kv", ops.lib().mivgpu_paged_qk_norm_rope_kv, _ptr(qkv),
            qkv.stride(0) if N > 1 else width, _ptr(q_norm_w), _ptr(k_norm_w), _ptr(positions), _ptr(slots), _ptr(turns),
            _ptr(q_out), _ptr(cache.k), _ptr(cache.v), _ptr(cache.k_scale), _ptr(cache.v_scale), N, n_q_heads, n_kv_heads,
            head_dim, pages, eps)
    return q_out


# -------------------------------------------------------------- attention --
def paged_attention_workspace(n_tokens: int, rows: int, n_q_heads: int, n_kv_heads: int, head_dim: int,
                              device="cuda") -> torch.Tensor:
    """Workspace of ``paged_attention`` for steps of up to ``n_tokens`` tokens and ``rows`` requests.  Calls that may
    run at once (two streams, two captured graphs replayed side by side) need one each."""
    return torch.empty(0, dtype=torch.float32, device=device)


def paged_attention(q: torch.Tensor, cache: PagedKV, table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor,
                    n_q_heads: int, n_kv_heads: int, head_dim: int, scale: float, max_new: int | None = None,
                    out: torch.Tensor | None = None, work: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention of packed tokens over their requests' pages -> out [N, Hq*D] bf16.

    q [N, Hq, D] bf16; request b owns rows cu_q[b] .. cu_q[b+1], the last of its kv_lens[b] positions; its pages are
    table[b] (int32 [B, W], B <= 1024).  A row that sees no key (a request with kv_lens 0) gives zeros; rows behind
    cu_q[B] are left as they are; keys on a page that the cache does not have count as masked.  ``max_new``: the most
    new tokens of a request, if known (1 in a decode step).  ``work`` from ``paged_attention_workspace``."""
    N = q.shape[0]
    B = kv_lens.numel()
    dev = q.device
    pages = _check_cache(cache, dev, "paged_attention", n_q_heads, n_kv_heads, head_dim)
    i32, bf = torch.int32, torch.bfloat16
    if out is None:
        out = torch.zeros(N, n_q_heads * head_dim, dtype=bf, device=dev)
    _on(dev, "paged_attention", q=(q, bf), table=(table, i32), cu_q=(cu_q, i32), kv_lens=(kv_lens, i32), out=(out, bf),
        work=(work, torch.float32))
    if tuple(q.shape) != (N, n_q_heads, head_dim) or tuple(out.shape) != (N, n_q_heads * head_dim):
        raise ValueError(f"paged_attention: q {tuple(q.shape)}, out {tuple(out.shape)} do not match {n_q_heads} heads of "
                         f"{head_dim}")
    if not 0 < B <= MAX_ROWS or tuple(kv_lens.shape) != (B,) or tuple(cu_q.shape) != (B + 1,) or table.dim() != 2 \
            or table.shape[0] != B or table.shape[1] < 1:
        raise ValueError(f"paged_attention: kv_lens [B <= {MAX_ROWS}], cu_q [B + 1], table [B, W]; got "
                         f"{tuple(kv_lens.shape)} {tuple(cu_q.shape)} {tuple(table.shape)}")
    if max_new is not None and max_new < 0:
        raise ValueError(f"paged_attention: max_new {max_new}")
    for what, t in (("q", q), ("out", out), ("k", cache.k), ("v", cache.v)):
        if N > 0 and t.data_ptr() % 16:
            raise ValueError(f"paged_attention: {what} must start at a multiple of 16 bytes")
    _launch(dev, "paged_attention", ops.lib().mivgpu_paged_attention, _ptr(q), _ptr(cache.k), _ptr(cache.v),
            _ptr(cache.k_scale), _ptr(cache.v_scale), _ptr(table), _ptr(cu_q), _ptr(kv_lens), _ptr(out), N, B,
            table.shape[1], n_q_heads, n_kv_heads, head_dim, pages, scale)
    return out
