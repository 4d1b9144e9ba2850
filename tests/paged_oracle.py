"""Plain 64-bit implementations of the paged 8-bit serving operators, for the tests: loops, on the host."""

import math

import numpy as np
import torch

PAGE = 64
EMIN, EMAX = -110, 119


def plan(new, lengths, table, free, ring, n_tokens):
    """Request by request, as one would by hand."""
    B, W = table.shape
    num = len(free)
    head, count = (int(x) for x in ring)
    table = table.copy()
    cu, kv, taken = [0], [], []
    positions, slots = np.zeros(n_tokens, np.int64), np.full(n_tokens, -1, np.int64)
    claimed = 0
    for b in range(B):
        n, have = max(int(new[b]), 0), -(-int(lengths[b]) // PAGE)
        total = int(lengths[b]) + n
        start = cu[-1]
        cu.append(start + n)
        fits = total <= PAGE * W and cu[-1] <= n_tokens
        need = -(-total // PAGE) - have if fits else 0
        first, claimed = claimed, claimed + need
        ok = fits and (need == 0 or claimed <= count)
        kv.append(total if ok else 0)
        taken.append(need if ok else -1)
        if ok:
            for j in range(need):
                table[b, have + j] = free[(head + first + j) % num]
            for i in range(n):
                p = int(lengths[b]) + i
                positions[start + i] = p
                slots[start + i] = int(table[b, p // PAGE]) * PAGE + p % PAGE
    return dict(cu_q=np.array(cu), kv_lens=np.array(kv), taken=np.array(taken), positions=positions, slots=slots, table=table)


def norm_rope(x, w, positions, theta, eps):
    """x [N, H, D] float64 -> (rotated, |a| + |b| of the pair behind each value)."""
    D = x.shape[-1]
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    # angles modulo a turn in extended precision: integer positions times a frequency, exact products of 53 x 32 bits
    f = [theta ** (-2.0 * i / D) for i in range(D // 2)]
    ang = torch.tensor([[math.fmod(float(np.longdouble(p) * np.longdouble(fi) % (2 * np.longdouble(np.pi))), 2 * math.pi)
                         for fi in f] for p in positions.tolist()], dtype=torch.float64).view(len(positions), 1, D // 2)
    c, s = torch.cos(ang), torch.sin(ang)
    a, b = x[..., :D // 2], x[..., D // 2:]
    size = a.abs() + b.abs()
    return torch.cat([a * c - b * s, b * c + a * s], -1), torch.cat([size, size], -1)


def scale_for(amax: float) -> float:
    """The smallest power of two with amax <= 448 * it."""
    e = EMIN
    while e < EMAX and amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def to_codes(x):
    """float64 -> e4m3, one rounding (float64 -> float32 first would be two: the values here are exact in float32)."""
    return x.clamp(-448, 448).to(torch.float32).to(torch.float8_e4m3fn)


def dequant(cache, side):
    """[pages, Hkv, 64, D] float64 of a cache (host tensors)."""
    if side == "k":
        return cache.k.to(torch.float32).double() * cache.k_scale.double()[..., None, None]
    return (cache.v.to(torch.float32).double() * cache.v_scale.double()[..., None, None]).transpose(-1, -2)


def attention(q, cache, table, cu, kv_lens, hq, hkv, scale):
    """-> (o [N, Hq, D] float64, mean |v| under the same weights, rows written); pages outside the cache are masked."""
    N, D = q.shape[0], q.shape[-1]
    k_all, v_all = dequant(cache, "k"), dequant(cache, "v")
    o, size = torch.zeros(N, hq, D, dtype=torch.float64), torch.zeros(N, hq, D, dtype=torch.float64)
    G, pages = hq // hkv, k_all.shape[0]
    for b in range(len(kv_lens)):
        s, e, L = int(cu[b]), min(int(cu[b + 1]), N), int(kv_lens[b])
        n = e - s
        if n <= 0 or L == 0:
            continue
        ids = torch.as_tensor(table[b, :-(-L // PAGE)]).long()
        ok = (ids >= 0) & (ids < pages)
        k = k_all[ids.clamp(0, pages - 1)].transpose(0, 1).reshape(hkv, -1, D)[:, :L]
        v = v_all[ids.clamp(0, pages - 1)].transpose(0, 1).reshape(hkv, -1, D)[:, :L]
        there = ok.repeat_interleave(PAGE)[:L]
        seen = (torch.arange(L)[None] <= (L - n + torch.arange(n))[:, None]) & there[None]
        for h in range(hq):
            sc = (q[s:e, h].double() @ k[h // G].T * scale).masked_fill(~seen, -math.inf)
            m = sc.amax(-1, keepdim=True)
            p = torch.where(seen, torch.exp(sc - torch.where(m.isinf(), torch.zeros_like(m), m)), torch.zeros_like(sc))
            t = p.sum(-1, keepdim=True)
            p = torch.where(t > 0, p / t, p)
            vh = torch.where(there[:, None], v[h // G], torch.zeros_like(v[h // G]))
            o[s:e, h] = p @ vh
            size[s:e, h] = p @ vh.abs()
    return o, size


def order(row, t, k, p, min_p):
    """A row's kept tokens in order and their weights (float64), for one row of float64 logits without NaN."""
    idx = np.lexsort((np.arange(len(row)), -row))
    idx = idx[row[idx] > -np.inf]
    if len(idx) == 0:
        return idx, np.zeros(0)
    if not t > 0:
        return idx[:1], np.ones(1)
    x = row[idx]
    w = np.where(x == x[0], 1.0, np.exp(np.where(x == x[0], 0.0, x - x[0]) / t))
    if k > 0:
        idx, w = idx[:k], w[:k]
    if p < 1:
        before = np.cumsum(w) - w
        n = max(1, int((before < p * w.sum()).sum()))
        idx, w = idx[:n], w[:n]
    n = max(1, int((w >= min_p).sum()))
    return idx[:n], w[:n]
