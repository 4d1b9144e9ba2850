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
import decimal
import math
from typing import NamedTuple

import torch

from k8s_vgpu_scheduler_amd import ops

PAGE = 64            # tokens of a page (csrc/ops/paged.h)
MAX_ROWS = 1024      # requests of one call
MAX_KV_HEADS = 256   # of paged_attention (csrc/ops/paged_attn.hip MAX_HKV)


_I32, _I64, _F32, _BF16, _FP8 = torch.int32, torch.int64, torch.float32, torch.bfloat16, torch.float8_e4m3fn


def _ptrs(name: str, *specs):
    """Device index and addresses of ``(what, tensor or None, dtype, shape)``: each contiguous, of its type and shape,
    all on one GPU.  (A fraction of a microsecond a tensor: a decode step makes these calls for every layer.)"""
    idx, out = None, []
    for what, t, dtype, shape in specs:
        if t is None:
            out.append(None)
            continue
        if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name}: {what} must be contiguous {dtype} {list(shape)}, got {t.dtype} {list(t.shape)} "
                             f"strides {list(t.stride())}")
        d = t.get_device()
        if d != idx:
            if idx is not None or d < 0:
                raise ValueError(f"{name}: {what} is on {t.device}: every tensor must be on one GPU")
            idx = d
        out.append(t.data_ptr())
    return idx, out


def _launch(idx: int, name: str, fn, *args):
    """The C call on the current stream of the tensors' GPU, whatever the current device is."""
    if idx == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    if rc == -2:
        raise ValueError(f"{name}: the workspace is too small for this call")
    if rc == -1:
        raise ValueError(f"{name}: sizes past the kernels' 32-bit indices")
    ops._check(rc, name)


def _misaligned(name: str, **ptrs):
    """Says which: the callers look at all addresses at once first."""
    for what, p in ptrs.items():
        if p % 16:
            raise ValueError(f"{name}: {what} must start at a multiple of 16 bytes")


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
    B, W = table.shape if table.dim() == 2 else (0, 0)
    pages = free.numel()
    if not 0 < B <= MAX_ROWS or W < 1 or free.dim() != 1 or pages < 1:
        raise ValueError(f"page_plan: table [B <= {MAX_ROWS}, W], free [pages], got {list(table.shape)} {list(free.shape)}")
    if n_tokens < 0 or max(pages, W) * PAGE > 2**31 - 1:
        raise ValueError(f"page_plan: n_tokens {n_tokens}, {pages} pages, {W} a request: slots are 32-bit")
    idx, p = _ptrs("page_plan", ("new_lens", new_lens, _I32, (B,)), ("lengths", lengths, _I32, (B,)),
                   ("table", table, _I32, (B, W)), ("free", free, _I32, (pages,)), ("ring", ring, _I32, (2,)))
    sizes = (B + 1, B, B, n_tokens, n_tokens)
    if out is None:
        buf = free.new_empty(sum(sizes))                                   # one allocation
        out = PagePlan(*torch.unsafe_split_with_sizes(buf, sizes))
        at = buf.data_ptr()
        for n in sizes:
            p.append(at)
            at += 4 * n
    else:
        on, more = _ptrs("page_plan", *((what, t, _I32, (n,)) for what, t, n in zip(PagePlan._fields, out, sizes)))
        if on != idx:
            raise ValueError("page_plan: every tensor must be on one GPU")
        p += more
    _launch(idx, "page_plan", ops.lib().mivgpu_page_plan, *p, B, W, pages, n_tokens)
    return out


def page_commit(plan: PagePlan, lengths: torch.Tensor, table: torch.Tensor, free: torch.Tensor, ring: torch.Tensor,
                finished: torch.Tensor | None = None):
    """The plan's step is done: ``lengths`` of admitted requests become its ``kv_lens`` and their pages leave the
    ring.  ``finished`` (bool [B]): requests whose pages go back to the ring's end, in order; their length becomes 0.  A plan
    is committed once."""
    if table.dim() != 2 or not 0 < table.shape[0] <= MAX_ROWS or table.shape[1] < 1 or free.dim() != 1 \
            or free.numel() < 1 or max(free.numel(), table.shape[1]) * PAGE > 2**31 - 1:
        raise ValueError(f"page_commit: table [B <= {MAX_ROWS}, W], free [pages], got {list(table.shape)} {list(free.shape)}")
    B, W = table.shape
    pages = free.numel()
    idx, p = _ptrs("page_commit", ("kv_lens", plan.kv_lens, _I32, (B,)), ("taken", plan.taken, _I32, (B,)),
                   ("finished", finished, torch.bool, (B,)), ("lengths", lengths, _I32, (B,)),
                   ("table", table, _I32, (B, W)), ("free", free, _I32, (pages,)), ("ring", ring, _I32, (2,)))
    _launch(idx, "page_commit", ops.lib().mivgpu_page_commit, *p, B, W, pages)


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
    k_scale, v_scale [pages, Hkv] fp32; a value is its code times its page's scale.  Scales are powers of two from
    2^-110 to 2^119: a query that sees a page with any other gives NaN."""
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


def _cache_specs(cache: PagedKV, name: str, n_q_heads: int, n_kv_heads: int, head_dim: int):
    """Host check of the head counts; the cache's pages and what ``_ptrs`` checks of it."""
    if n_kv_heads < 1 or n_q_heads < 1 or n_q_heads % n_kv_heads or head_dim not in (64, 128):
        raise ValueError(f"{name}: {n_q_heads} / {n_kv_heads} heads of {head_dim} (64 or 128)")
    pages = cache.k.shape[0]
    if pages < 1 or pages * PAGE > 2**31 - 1:
        raise ValueError(f"{name}: {pages} pages: slots are 32-bit")
    return pages, (("k", cache.k, _FP8, (pages, n_kv_heads, PAGE, head_dim)),
                   ("v", cache.v, _FP8, (pages, n_kv_heads, head_dim, PAGE)),
                   ("k_scale", cache.k_scale, _F32, (pages, n_kv_heads)),
                   ("v_scale", cache.v_scale, _F32, (pages, n_kv_heads)))


# ----------------------------------------------------------------- append --
_PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def rope_turns(theta: float, head_dim: int, device="cuda") -> torch.Tensor:
    """The rotation's table: 2^64 * theta^(-2i/D) / 2pi for i < D/2, rounded (int64 bits).  A position's angle in
    turns is the fraction position * turns / 2^64, exact to 2^-65 of the position (so the entries are computed to 60
    digits: from 64-bit floats they are off by hundreds of their last place)."""
    if head_dim not in (64, 128) or not 1 <= theta < math.inf:
        raise ValueError(f"rope_turns: theta {theta} (at least 1), head_dim {head_dim} (64 or 128)")
    vals = []
    with decimal.localcontext(decimal.Context(prec=60, rounding=decimal.ROUND_HALF_EVEN)):
        x, step = 2**63 / _PI, decimal.Decimal(float(theta)) ** (decimal.Decimal(-2) / head_dim)
        for _ in range(head_dim // 2):
            vals.append(int(x.to_integral_value()))
            x *= step
    return torch.tensor(vals, dtype=torch.int64, device=device)      # at most 2^64 / 2pi < 2^63


def paged_qk_norm_rope_kv(qkv: torch.Tensor, q_norm_w: torch.Tensor, k_norm_w: torch.Tensor, positions: torch.Tensor,
                          slots: torch.Tensor, turns: torch.Tensor, cache: PagedKV, q_out: torch.Tensor, n_q_heads: int,
                          n_kv_heads: int, head_dim: int, eps: float):
    """Packed tokens qkv [N, (Hq+2Hkv)*D] bf16 (rows may be strided, by a multiple of 8) -> per-head RMSNorm of q and
    k, NeoX RoPE at ``positions`` [N] -> q_out [N, Hq, D] bf16; K and V appended to ``cache`` at ``slots`` [N].

    A row whose slot is outside the cache appends nothing (its q_out is written).  Tokens of one page stand together,
    in the order of their slots, behind the page's live tokens: a page whose first slot is written starts afresh, any
    other keeps its earlier tokens, whose codes follow when a new value raises the page's scale.  (``PagePool.plan``
    gives such slots.)  A token whose K or V of a head is not finite is stored as NaN in K and zero in V."""
    name = "paged_qk_norm_rope_kv"
    pages, specs = _cache_specs(cache, name, n_q_heads, n_kv_heads, head_dim)
    width = (n_q_heads + 2 * n_kv_heads) * head_dim
    N = positions.shape[0] if positions.dim() == 1 else -1
    ld, one = qkv.stride() if qkv.dim() == 2 else (0, 0)
    if qkv.dtype is not _BF16 or qkv.shape != (N, width) or (N > 0 and one != 1) or (N > 1 and (ld % 8 or ld < width)):
        raise ValueError(f"{name}: qkv must be bf16 [{N}, {width}] with unit column stride and a row stride that is a "
                         f"multiple of 8, got {qkv.dtype} {list(qkv.shape)} strides {list(qkv.stride())}")
    idx, p = _ptrs(name, ("q_norm_w", q_norm_w, _BF16, (head_dim,)), ("k_norm_w", k_norm_w, _BF16, (head_dim,)),
                   ("positions", positions, _I32, (N,)), ("slots", slots, _I32, (N,)),
                   ("turns", turns, _I64, (head_dim // 2,)), ("q_out", q_out, _BF16, (N, n_q_heads, head_dim)), *specs)
    if qkv.get_device() != idx:
        raise ValueError(f"{name}: qkv is on {qkv.device}: every tensor must be on one GPU")
    x = qkv.data_ptr()
    if (x | p[0] | p[1] | p[5] | p[6] | p[7]) & 15:
        _misaligned(name, qkv=x, q_norm_w=p[0], k_norm_w=p[1], q_out=p[5], k=p[6], v=p[7])
    _launch(idx, name, ops.lib().mivgpu_paged_qk_norm_rope_kv, x, ld if N > 1 else width, *p, N, n_q_heads, n_kv_heads,
            head_dim, pages, eps)
    return q_out


# -------------------------------------------------------------- attention --
def paged_attention_workspace(n_tokens: int, rows: int, n_q_heads: int, n_kv_heads: int, head_dim: int,
                              device="cuda") -> torch.Tensor:
    """Workspace of ``paged_attention`` for steps of up to ``n_tokens`` tokens and ``rows`` requests: room for the parts
    that a long request is split into, and counters that every call leaves at zero.  Calls that may run at once (two
    streams, two captured graphs replayed side by side) need one each."""
    if not 0 <= n_tokens < 2**31 or not 0 < rows <= MAX_ROWS or not 0 < n_kv_heads <= MAX_KV_HEADS or n_q_heads < 1 \
            or n_q_heads % n_kv_heads or head_dim not in (64, 128):
        raise ValueError(f"paged_attention_workspace: {n_tokens} tokens of {rows} requests, {n_q_heads} / {n_kv_heads} "
                         f"(at most {MAX_KV_HEADS}) heads of {head_dim} (64 or 128)")
    zeroed = ctypes.c_longlong(0)
    with torch.cuda.device(device):
        floats = ops.lib().mivgpu_paged_attention_work(n_tokens, n_q_heads, n_kv_heads, ctypes.byref(zeroed))
    work = torch.empty(floats, dtype=_F32, device=device)
    work[:zeroed.value].zero_()
    return work


def paged_attention(q: torch.Tensor, cache: PagedKV, table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor,
                    n_q_heads: int, n_kv_heads: int, head_dim: int, scale: float, max_new: int | None = None,
                    out: torch.Tensor | None = None, work: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention of packed tokens over their requests' pages -> out [N, Hq*D] bf16.

    q [N, Hq, D] bf16; request b owns rows cu_q[b] .. cu_q[b+1], the last of its kv_lens[b] positions (at most 64 W); its
    pages are table[b] (int32 [B, W], B <= 1024).  A row that sees no key (a request with kv_lens 0) gives zeros; rows
    behind cu_q[B] are left as they are; keys on a page that the cache does not have count as masked.  ``max_new``: the
    most new tokens of a request, if known (1 in a decode step, which is then faster for many requests).  ``work`` from
    ``paged_attention_workspace``."""
    name = "paged_attention"
    pages, specs = _cache_specs(cache, name, n_q_heads, n_kv_heads, head_dim)
    if n_kv_heads > MAX_KV_HEADS:
        raise ValueError(f"{name}: {n_kv_heads} kv heads (at most {MAX_KV_HEADS})")
    if q.dim() != 3 or not 2.0 ** -126 <= scale <= 2.0 ** 126:      # a normal fp32 number, times log2(e) too
        raise ValueError(f"{name}: q must be [N, {n_q_heads}, {head_dim}], got {list(q.shape)}, and scale in "
                         f"2^-126 .. 2^126, got {scale}")
    N = q.shape[0]
    B, W = table.shape if table.dim() == 2 else (0, 0)
    if not 0 < B <= MAX_ROWS or not 0 < W <= (2**31 - 1) // PAGE:
        raise ValueError(f"{name}: table must be [B <= {MAX_ROWS}, W], got {list(table.shape)}")
    if max_new is not None and not 0 <= max_new < 2**31:
        raise ValueError(f"{name}: max_new {max_new}")
    if out is None:
        out = torch.zeros(N, n_q_heads * head_dim, dtype=_BF16, device=q.device)
    idx, p = _ptrs(name, ("q", q, _BF16, (N, n_q_heads, head_dim)), *specs, ("table", table, _I32, (B, W)),
                   ("cu_q", cu_q, _I32, (B + 1,)), ("kv_lens", kv_lens, _I32, (B,)),
                   ("out", out, _BF16, (N, n_q_heads * head_dim)))
    if work is None:
        work = paged_attention_workspace(N, B, n_q_heads, n_kv_heads, head_dim, q.device)
    if work.dtype is not _F32 or work.dim() != 1 or not work.is_contiguous() or work.get_device() != idx:
        raise ValueError(f"{name}: work must be from paged_attention_workspace on {q.device}")
    room = work.data_ptr()
    if (p[0] | p[1] | p[2] | p[8] | room) & 15:
        _misaligned(name, q=p[0], k=p[1], v=p[2], out=p[8], work=room)
    _launch(idx, name, ops.lib().mivgpu_paged_attention, *p, room, work.numel(), N, B, W, n_q_heads, n_kv_heads,
            head_dim, pages, -1 if max_new is None else max_new, scale)
    return out
