"""What the paged 8-bit serving operators are measured on: the cases, their inputs, the plain forms and the
framework's calls.

Four operators, in the order in which a serving step uses them:

  plan    pages for the new tokens of a batch of requests: block tables, slot map, positions, key counts
  append  QK-norm + RoPE over a ragged batch of tokens, K/V appended to 8-bit pages (e4m3, one power-of-two
          scale for each page and head)
  attn    attention of the new tokens over the pages: single tokens, chunks of a prompt, whole prompts
  sample  a token for each row of logits: temperature, top-k, top-p, min-p, from given random numbers

``run`` computes the plain form (elementary torch operations) unless ``own`` is set; then it makes the framework's
calls.  ``exact`` follows the definitions in 64 bits.
"""

import math

import numpy as np
import torch

own = False

PAGE = 64                    # tokens of a page
EMIN, EMAX = -110, 119       # exponents of a page's scale
E4M3_MAX = 448.0
EPS, THETA = 1e-6, 1e6
VOCAB = 151936


def listed():
    return [
        # a decode step's pages: 32 running requests, one new token each
        dict(name="plan decode 32", op="plan", rows=32, new=1, longs=0, long_new=0, ctx=8192),
        # a step that mixes four prompts of about 2000 tokens with 252 running requests
        dict(name="plan mixed 256", op="plan", rows=256, new=1, longs=4, long_new=2000, ctx=8192),
        # K/V of a decode step: the headline decode batch
        dict(name="append decode 32", op="append", rows=32, new=1, longs=0, long_new=0, ctx=1024, hq=32, hkv=8, d=128),
        # K/V of a prompt as long as the server takes them, in one pass
        dict(name="append prompt 8192", op="append", rows=1, new=8192, longs=0, long_new=0, ctx=0, hq=32, hkv=8, d=128),
        # one user, late in a long conversation: a single row against 8191 keys
        dict(name="attn single 8191", op="attn", rows=1, new=1, longs=0, long_new=0, ctx=8190, ragged=False, hq=32, hkv=8, d=128),
        # the headline decode batch: 32 rows of about 1000 keys
        dict(name="attn decode 32x1024", op="attn", rows=32, new=1, longs=0, long_new=0, ctx=1024, ragged=False, hq=32, hkv=8, d=128),
        # a busy server: 64 rows from a few keys to 32768, narrow heads in groups of eight
        dict(name="attn decode ragged", op="attn", rows=64, new=1, longs=0, long_new=0, ctx=32768, ragged=True, hq=32, hkv=4, d=64),
        # a chunk of a prompt behind 4096 cached tokens, beside seven running requests
        dict(name="attn chunk mixed", op="attn", rows=8, new=1, longs=1, long_new=1000, ctx=4096, ragged=True, hq=32, hkv=8, d=128),
        # a whole prompt as long as the server takes them
        dict(name="attn prompt 8192", op="attn", rows=1, new=8192, longs=0, long_new=0, ctx=0, ragged=False, hq=32, hkv=8, d=128),
        # the next token of one stream: latency
        dict(name="sample 1", op="sample", rows=1, vocab=VOCAB, mix=False),
        # the headline decode batch, each request with settings of its own
        dict(name="sample 32", op="sample", rows=32, vocab=VOCAB, mix=True),
        # the largest decode batch
        dict(name="sample 256", op="sample", rows=256, vocab=VOCAB, mix=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attn", "attn", "sample"])
    heads = rng.choice([(32, 8, 128), (8, 2, 128), (12, 2, 128), (16, 16, 128), (32, 4, 64), (32, 2, 128), (8, 8, 64)])
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, VOCAB), mix=rng.random() < 0.75)
    if op == "attn":
        hq, hkv, d = heads
        if rng.random() < 0.6:      # rows of one or a few new tokens
            return dict(op=op, rows=_log(rng, 1, 64), new=rng.choice([1, 1, 1, 2, 5]), longs=0, long_new=0,
                        ctx=_log(rng, 1, 32768 * 4 // max(4, hkv)), ragged=rng.random() < 0.7, hq=hq, hkv=hkv, d=d)
        return dict(op=op, rows=rng.randint(1, 4), new=1, longs=1, long_new=_log(rng, 17, 4096), ctx=_log(rng, 1, 4096),
                    ragged=True, hq=hq, hkv=hkv, d=d)
    case = dict(op=op, rows=_log(rng, 1, 256), new=rng.choice([1, 1, 3]), longs=0, long_new=0, ctx=_log(rng, 1, 8192))
    if rng.random() < 0.5:
        case["longs"] = min(rng.randint(1, 3), case["rows"])
        case["long_new"] = _log(rng, 17, 2400)
    if op == "append":
        case["hq"], case["hkv"], case["d"] = heads
    return case


# ------------------------------------------------------------------ inputs --
def _lens(case, seed):
    """Tokens cached and new of each request: the case says which lengths, the seed in which order."""
    r = np.random.RandomState(case["rows"] * 7919 + case["ctx"])
    B, ctx = case["rows"], case["ctx"]
    if ctx == 0:
        old = np.zeros(B, dtype=np.int64)
    elif case.get("ragged", True):
        old = np.exp(r.uniform(0, math.log(ctx), B)).astype(np.int64)
        old[r.randint(B)] = ctx
    else:
        old = ctx + r.randint(-(ctx // 64), 1, B) if B > 1 else np.array([ctx])
    new = np.full(B, case["new"], dtype=np.int64)
    for b in r.permutation(B)[:case["longs"]]:
        new[b] = max(1, int(case["long_new"] * r.uniform(0.85, 1.0)))
        old[b] = ctx
    order = np.random.RandomState(seed).permutation(B)
    return old[order], new[order]


def _pages(old, new, r, spare):
    """Distinct pages of a shuffled pool for the cached tokens and, behind them, `spare` free ones."""
    have = -(-old // PAGE)
    total = int(have.sum()) + spare
    pool = r.permutation(total).astype(np.int32)
    width = int((-(-(old + new) // PAGE)).max())
    table = np.full((len(old), width), -1, dtype=np.int32)
    at = 0
    for b, h in enumerate(have):
        table[b, :h] = pool[at:at + h]
        at += int(h)
    return table, pool[at:], total


def _step(old, new, seed):
    """The layout of a step: every request with pages for its cached and its new tokens."""
    r = np.random.RandomState(seed + 1)
    table, free, total = _pages(old + new, new * 0, r, 3)
    cu = np.concatenate([[0], np.cumsum(new)])
    b = np.repeat(np.arange(len(new)), new)
    pos = old[b] + np.arange(cu[-1]) - cu[b]
    slots = table[b, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()  # noqa: E731
    return dict(table=dev(table), cu_q=dev(cu), kv_lens=dev(old + new), positions=dev(pos), slots=dev(slots), pages=total)


def _cache(pages, hkv, d, g):
    """Filled pages: keys and values of unit size, as codes and a power-of-two scale for each page and head."""
    def side(shape):
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
        e = torch.randint(-8, -6, (pages, hkv), generator=g, device="cuda", dtype=torch.int32)
        s = ((e + 127) << 23).view(torch.float32)
        return (x / s[:, :, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), s

    k, ks = side((pages, hkv, PAGE, d))
    v, vs = side((pages, hkv, d, PAGE))
    return dict(k=k, v=v, k_scale=ks, v_scale=vs)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    if op == "sample":
        B, V = case["rows"], case["vocab"]
        # logits of a language model: a broad bulk and a few likely tokens; a tenth of the rows have a vocabulary mask
        x = torch.randn(B, V, generator=g, device="cuda") * 2.2
        top = torch.randint(0, V, (B, 24), generator=g, device="cuda")
        x.scatter_add_(1, top, torch.rand(B, 24, generator=g, device="cuda") * 14)
        banned = torch.rand(B, V, generator=g, device="cuda") < 0.3
        some = torch.rand(B, 1, generator=g, device="cuda") < 0.1
        logits = x.masked_fill(banned & some, float("-inf")).to(torch.bfloat16)
        u = torch.rand(B, generator=g, device="cuda")
        r = np.random.RandomState(seed)
        if case["mix"]:
            t = r.choice([0.0, 0.6, 0.7, 0.8, 1.0, 1.3], B)
            k, p, mp = r.choice([0, 0, 20, 50, 1000], B), r.choice([1.0, 0.8, 0.9, 0.95], B), r.choice([0.0, 0.0, 0.02, 0.1], B)
        else:
            t, k, p, mp = np.full(B, 0.7), np.full(B, 0), np.full(B, 0.95), np.full(B, 0.0)
        f = lambda a, dt: torch.tensor(a, dtype=dt, device="cuda")  # noqa: E731
        state = dict(op=op, logits=logits, u=u, t=f(t, torch.float32), k=f(k, torch.int32), p=f(p, torch.float32),
                     min_p=f(mp, torch.float32))
        if own:
            from k8s_vgpu_scheduler_amd import ops
            state["work"] = ops.sample_workspace(B, V, "cuda")
        return state
    old, new = _lens(case, seed)
    if op == "plan":
        r = np.random.RandomState(seed + 1)
        need = int((-(-(old + new) // PAGE) - -(-old // PAGE)).sum())
        # most steps find enough free pages; every fourth input runs out for the last requests
        count = need + 9 if seed % 4 else max(1, need - 2)
        table, free, total = _pages(old, new, r, count)
        ring = np.zeros(total, dtype=np.int32)
        head = int(r.randint(total))
        ring[(head + np.arange(len(free))) % total] = free
        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()  # noqa: E731
        return dict(op=op, new=dev(new), lengths=dev(old), table=dev(table), free=dev(ring), ring=dev([head, count]),
                    n_tokens=int(new.sum()))
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    step = _step(old, new, seed)
    N = int(new.sum())
    state = dict(op=op, hq=hq, hkv=hkv, d=d, n=N, max_new=int(new.max()), max_len=int((old + new).max()),
                 **step, **_cache(step["pages"], hkv, d, g))
    if op == "append":
        state["qkv"] = (torch.randn(N, (hq + 2 * hkv) * d, generator=g, device="cuda")
                        * (0.5 + 1.5 * torch.rand((hq + 2 * hkv) * d, generator=g, device="cuda"))).to(torch.bfloat16)
        w = lambda: (1 + 0.05 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)  # noqa: E731
        state["qw"], state["kw"] = w(), w()
        state["q_out"] = torch.empty(N, hq, d, dtype=torch.bfloat16, device="cuda")
        if own:
            from k8s_vgpu_scheduler_amd import ops
            state["turns"] = ops.rope_turns(THETA, d, "cuda")
    else:
        state["q"] = torch.randn(N, hq, d, generator=g, device="cuda").to(torch.bfloat16)
        state["out"] = torch.empty(N, hq * d, dtype=torch.bfloat16, device="cuda")
        if own:
            from k8s_vgpu_scheduler_amd import ops
            state["work"] = ops.paged_attention_workspace(N, len(new), hq, hkv, d, "cuda")
    return state


# ------------------------------------------------------------- plain forms --
def _plain_plan(s):
    length, table, free = s["lengths"].long(), s["table"], s["free"]
    B, W = table.shape
    N, num = s["n_tokens"], free.numel()
    head, count = s["ring"][0].long(), s["ring"][1].long()
    n = s["new"].clamp(min=0).long()
    end = torch.cumsum(n, 0)
    total = length + n
    have = (length + PAGE - 1) // PAGE
    fits = (total <= PAGE * W) & (end <= N)
    need = torch.where(fits, (total + PAGE - 1) // PAGE - have, 0)
    cum = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (cum <= count))
    i = torch.arange(N, device=length.device)
    b = torch.searchsorted(end, i, right=True)
    live = b < B
    b = b.clamp(max=B - 1)
    live &= ok[b]
    pos = torch.where(live, length[b] + i - (end - n)[b], 0)
    j = pos // PAGE
    fresh = free[(head + (cum - need)[b] + j - have[b]) % num].long()
    page = torch.where(j < have[b], table[b, j].long(), fresh)
    slots = torch.where(live, page * PAGE + pos % PAGE, -1)
    flat = torch.cat([table.view(-1), table.new_zeros(1)])
    flat[torch.where(live, b * W + j, B * W)] = page.int()
    table.copy_(flat[:-1].view(B, W))
    cu = torch.cat([end.new_zeros(1), end])
    return dict(cu_q=cu.int(), kv_lens=torch.where(ok, total, 0).int(), taken=torch.where(ok, need, -1).int(),
                positions=pos.int(), slots=slots.int(), table=table)


def _scale_of(amax):
    m, x = torch.frexp(amax)
    e = torch.where(amax > 0, x - 9 + (m > 0.875).int(), EMIN).clamp(EMIN, EMAX)
    return ((e.int() + 127) << 23).view(torch.float32)


def _rotated(s, x, w):
    """RMS norm over each head, then the rotation of its halves; angles in 64 bits."""
    d = s["d"]
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    freq = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d)
    a = s["positions"].double()[:, None] * freq
    c, sn = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1)


def _plain_append(s):
    N, hq, hkv, d = s["n"], s["hq"], s["hkv"], s["d"]
    x = s["qkv"].float().view(N, hq + 2 * hkv, d)
    q, k, v = _rotated(s, x[:, :hq], s["qw"]), _rotated(s, x[:, hq:hq + hkv], s["kw"]), x[:, hq + hkv:]
    slots = s["slots"].long()
    page, off = slots // PAGE, slots % PAGE
    bad = ~(k.isfinite().all(-1) & v.isfinite().all(-1))
    k, v = k.masked_fill(bad[..., None], float("nan")), v.masked_fill(bad[..., None], 0.0)
    at = torch.full((s["pages"],), PAGE, dtype=torch.long, device=x.device).scatter_reduce(0, page, off, "amin")
    touched, fresh = (at < PAGE)[:, None], (at == 0)[:, None]
    older = torch.arange(PAGE, device=x.device) < at[:, None]           # live tokens of a page from before
    older &= touched
    new = {}
    for name, val in (("k", k), ("v", v)):
        amax = torch.zeros(s["pages"], hkv, device=x.device).scatter_reduce(
            0, page[:, None].expand(N, hkv), val.abs().amax(-1).nan_to_num(0.0), "amax")
        before = s[name + "_scale"]
        made = _scale_of(amax)
        scale = torch.where(touched, torch.where(fresh, made, torch.maximum(made, before)), before)
        live = older[:, None, :, None] if name == "k" else older[:, None, None, :]
        codes = s[name]
        old = (codes.float() * (before / scale)[:, :, None, None]).to(torch.float8_e4m3fn)
        bits = torch.where(live, old.view(torch.uint8), codes.view(torch.uint8))
        fit = (val / scale[page][..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
        if name == "k":
            bits[page, :, off] = fit
        else:
            bits[page, :, :, off] = fit
        s[name].view(torch.uint8).copy_(bits)
        before.copy_(scale)
    return dict(q=q.to(torch.bfloat16), k=s["k"], v=s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _plain_attn(s):
    hq, hkv, d, n, L = s["hq"], s["hkv"], s["d"], s["max_new"], s["max_len"]
    cu, kv = s["cu_q"].long(), s["kv_lens"].long()
    B, G, W = kv.numel(), hq // hkv, -(-L // PAGE)
    pages = s["table"][:, :W].clamp(min=0).long()
    k = s["k"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s["k_scale"][pages][..., None, None]
    k = k.transpose(1, 2).reshape(B, hkv, W * PAGE, d)
    v = s["v"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s["v_scale"][pages][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(B, hkv, W * PAGE, d)
    i = torch.arange(n, device=kv.device)
    mine = i < (cu[1:] - cu[:-1])[:, None]                                    # [B, n]
    row = (cu[:-1, None] + i).clamp(max=s["n"] - 1)
    q = s["q"].float()[row].view(B, n, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * n, d)
    pos = (kv - (cu[1:] - cu[:-1]))[:, None] + i
    key = torch.arange(W * PAGE, device=kv.device)
    seen = (key <= pos[..., None]) & (key < kv[:, None, None])                # [B, n, keys]
    sc = torch.matmul(q, k.transpose(-1, -2)).view(B, hkv, G, n, W * PAGE) / math.sqrt(d)
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc.sub_(torch.where(m.isinf(), 0.0, m)))
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill((key >= kv[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.view(B, hkv, G * n, W * PAGE), v).view(B, hkv, G, n, d) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, hq * d)
    return o[mine].to(torch.bfloat16)


def _plain_sample(s):
    x, order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    t = s["t"].double()[:, None]
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    V = x.shape[-1]
    rank = torch.arange(V, device=x.device)
    k = torch.where(t > 0, torch.where(s["k"] > 0, s["k"], V)[:, None], 1)
    w = torch.where(rank < k, w, 0.0)
    c = torch.cumsum(w, -1)
    p = s["p"].double()[:, None]
    w = torch.where(((c - w) < p * c[:, -1:]) | (p >= 1) | (rank == 0), w, 0.0)
    w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    c = torch.cumsum(w, -1)
    last = (w > 0).sum(-1, keepdim=True) - 1
    at = torch.minimum((c <= s["u"].double()[:, None] * c[:, -1:]).sum(-1, keepdim=True), last)
    return dict(tokens=order.gather(-1, at)[:, 0], probs=(w.gather(-1, at) / c[:, -1:])[:, 0].float())


_PLAIN = dict(plan=_plain_plan, append=_plain_append, attn=_plain_attn, sample=_plain_sample)


def run(state):
    if not own:
        return _PLAIN[state["op"]](state)
    from k8s_vgpu_scheduler_amd import ops
    s = state
    if s["op"] == "plan":
        p = ops.page_plan(s["new"], s["lengths"], s["table"], s["free"], s["ring"], s["n_tokens"])
        return dict(cu_q=p.cu_q, kv_lens=p.kv_lens, taken=p.taken, positions=p.positions, slots=p.slots, table=s["table"])
    if s["op"] == "sample":
        tokens, probs = ops.sample(s["logits"], s["u"], s["t"], s["k"], s["p"], s["min_p"], work=s["work"])
        return dict(tokens=tokens, probs=probs)
    cache = ops.PagedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["op"] == "append":
        ops.paged_qk_norm_rope_kv(s["qkv"], s["qw"], s["kw"], s["positions"], s["slots"], s["turns"], cache, s["q_out"],
                                  s["hq"], s["hkv"], s["d"], EPS)
        return dict(q=s["q_out"], k=s["k"], v=s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return ops.paged_attention(s["q"], cache, s["table"], s["cu_q"], s["kv_lens"], s["hq"], s["hkv"], s["d"],
                               1.0 / math.sqrt(s["d"]), max_new=s["max_new"], out=s["out"], work=s["work"])


# -------------------------------------------------------------------- work --
def work(case):
    op = case["op"]
    if op == "sample":      # the logits once, a compare and a count each; the row's settings and its answer
        n = case["rows"] * case["vocab"]
        return dict(bytes=2 * n + case["rows"] * 32, flops=2 * n)
    old, new = _lens(case, 1)
    N, B = int(new.sum()), len(new)
    if op == "plan":        # lengths in and out, the table's new entries, a slot and a position for each token
        pages = int((-(-(old + new) // PAGE)).sum())
        return dict(bytes=4 * (5 * B + 2 * N + pages + N // PAGE), flops=8 * N)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if op == "append":      # the rows in, q out, a byte for each K and V value
        return dict(bytes=N * d * (2 * (hq + 2 * hkv) + 2 * hq + 2 * hkv), flops=N * d * (hq + hkv) * 10)
    pairs = float((new * old + new * (new + 1) // 2).sum())
    return dict(bytes=2 * float((old + new).sum()) * hkv * d + 4 * N * hq * d, flops=4 * pairs * hq * d)


# ------------------------------------------------------------------- exact --
def _exact_sample(s):
    x = s["logits"].double().cpu().numpy()
    u, t, k = (s[n].double().cpu().numpy() for n in ("u", "t", "k"))
    p, mp = (s[n].double().cpu().numpy() for n in ("p", "min_p"))
    probs = np.empty(len(x))
    for b, row in enumerate(x):
        if t[b] <= 0:
            probs[b] = 1.0
            continue
        y = np.sort(row)[::-1]
        w = np.exp((y - y[0]) / t[b])
        if 0 < k[b] < len(w):
            w = w[:int(k[b])]
        if p[b] < 1:
            w = w[:max(1, int(np.searchsorted(np.cumsum(w), p[b] * w.sum(), side="left")) + 1)]
        w = w[w >= mp[b]]
        c = np.cumsum(w)
        at = min(int(np.searchsorted(c, u[b] * c[-1], side="right")), int((w > 0).sum()) - 1)
        probs[b] = w[at] / c[-1]
    return dict(tokens=None, probs=torch.from_numpy(probs))


def _exact_append(s):
    """q in 64 bits; the pages' new codes before their rounding, the others as they stand; scales from the page's
    largest value."""
    N, hq, hkv, d = s["n"], s["hq"], s["hkv"], s["d"]
    x = s["qkv"].double().view(N, hq + 2 * hkv, d)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"),
                                                                    -2.0 / d * torch.arange(d // 2, device="cuda")))

    def rot(y, w):
        y = y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        z = torch.complex(y[..., :d // 2], y[..., d // 2:]) * turn[:, None]
        return torch.cat([z.real, z.imag], -1)

    q, k, v = rot(x[:, :hq], s["qw"]), rot(x[:, hq:hq + hkv], s["kw"]), x[:, hq + hkv:]
    slots = s["slots"].cpu().numpy()
    cache = {n: s[n].double() for n in ("k", "v", "k_scale", "v_scale")}
    first = np.flatnonzero(np.r_[True, slots[1:] // PAGE != slots[:-1] // PAGE])
    for a, z in zip(first, np.r_[first[1:], N]):
        page, lo, hi = slots[a] // PAGE, slots[a] % PAGE, slots[z - 1] % PAGE + 1
        for name, val in (("k", k[a:z]), ("v", v[a:z])):
            made = torch.exp2(torch.ceil(torch.log2(val.abs().amax((0, 2)) / E4M3_MAX)).clamp(EMIN, EMAX))
            sc = cache[name + "_scale"]
            now = torch.maximum(made, sc[page]) if lo else made
            c = cache[name][page]
            if name == "k":
                c[:, :lo] *= (sc[page] / now)[:, None, None]
                c[:, lo:hi] = (val / now[:, None]).transpose(0, 1)
            else:
                c[:, :, :lo] *= (sc[page] / now)[:, None, None]
                c[:, :, lo:hi] = (val / now[:, None]).permute(1, 2, 0)
            sc[page] = now
    return dict(q=q, **cache)


def _exact_attn(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    G = hq // hkv
    cu, kv = s["cu_q"].tolist(), s["kv_lens"].tolist()
    out = torch.zeros(s["n"], hq, d, dtype=torch.float64, device="cuda")
    for b, L in enumerate(kv):
        n = cu[b + 1] - cu[b]
        ids = s["table"][b, :-(-L // PAGE)].long()
        for h in range(hkv):
            k = (s["k"][:, h].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
                 * s["k_scale"][ids, h].double()[:, None, None]).reshape(-1, d)[:L]
            v = (s["v"][:, h].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
                 * s["v_scale"][ids, h].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:L]
            for g in range(G):
                a = s["q"][cu[b]:cu[b + 1], h * G + g].double() @ k.T / d ** 0.5
                if n > 1:
                    a += torch.full((n, L), -math.inf, dtype=torch.float64, device="cuda").triu(L - n + 1)
                out[cu[b]:cu[b + 1], h * G + g] = torch.softmax(a, -1) @ v
    return out.view(s["n"], hq * d)


def exact(case, seed):
    if case["op"] == "plan":
        return None         # whole numbers
    return dict(append=_exact_append, attn=_exact_attn, sample=_exact_sample)[case["op"]](prepare(case, seed))
