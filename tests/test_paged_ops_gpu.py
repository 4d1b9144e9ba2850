"""The paged 8-bit serving operators on the GPU against plain 64-bit implementations (tests/paged_oracle.py)."""

import ctypes
import math

import numpy as np
import paged_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE, THETA, EPS = 64, 1e6, 1e-6


@pytest.fixture(scope="module")
def ops():
    from k8s_vgpu_scheduler_amd import ops as o
    from k8s_vgpu_scheduler_amd.utils import build

    build.build_ops()
    o.require_native()
    return o


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(x)).to(dtype).cuda()


def host(t):
    return t.cpu().numpy()


# ------------------------------------------------------------------- plan --
def pool_state(lengths, width, spare, seed):
    """A table with distinct pages for `lengths`, and a ring with `spare` free ones behind."""
    r = np.random.RandomState(seed)
    have = -(-np.asarray(lengths) // PAGE)
    num = int(have.sum()) + spare + 2
    ids = r.permutation(num)
    table = np.full((len(lengths), width), -7)
    at = 0
    for b, h in enumerate(have):
        table[b, :h] = ids[at:at + h]
        at += h
    head = int(r.randint(num))
    ring = np.zeros(num, np.int64)
    ring[(head + np.arange(num - at)) % num] = ids[at:]
    return table, ring, [head, spare]


PLANS = {
    "one token": ([1], [0], 4, 1, 9),
    "nothing new": ([0, 0], [3, 0], 2, 0, 5),
    "no tokens, no rows": ([0], [0], 1, 0, 0),
    "page border": ([1, 1, 1, 64, 65], [63, 64, 65, 0, 0], 4, 20, 132),
    "padded rows": ([3, 0, 2], [10, 5, 0], 3, 9, 40),
    "out of pages": ([70, 65, 1, 200], [10, 0, 3, 0], 8, 3, 400),
    "refused, then one that needs none": ([65, 130, 1], [0, 0, 3], 8, 2, 400),
    "wider than the table": ([200, 64], [0, 64], 2, 9, 400),
    "more tokens than rows": ([50, 60, 5], [0, 0, 0], 4, 9, 112),
    "negative counts as none": ([-5, 3], [7, 0], 2, 4, 3),
    "ring empty": ([1, 1], [64, 3], 4, 0, 2),
}


@pytest.mark.parametrize("case", PLANS, ids=list(PLANS))
def test_plan(ops, case):
    new, old, width, spare, n = PLANS[case]
    check_plan(ops, new, old, width, spare, n, seed=3)


@pytest.mark.parametrize("rows,tokens,seed", [(32, 1, 1), (256, 40, 2), (1000, 3, 3), (1024, 9, 4), (5, 9000, 5)])
def test_plan_many(ops, rows, tokens, seed):
    r = np.random.RandomState(seed)
    new, old = r.randint(0, tokens + 1, rows), r.randint(0, 5000, rows)
    need = int((-(-(old + new) // PAGE) - -(-old // PAGE)).sum())
    for spare in (need, max(0, need - 3)):
        check_plan(ops, new, old, -(-int((old + new).max()) // PAGE), spare, int(new.sum()) + 7, seed)


def check_plan(ops, new, old, width, spare, n, seed):
    table, free, ring = pool_state(old, width, spare, seed)
    t, f, rg, ln, nw = dev(table), dev(free), dev(ring), dev(old), dev(new)
    want = oracle.plan(new, old, table, free, ring, n)
    for _ in range(2):                                   # planning again changes nothing
        got = ops.page_plan(nw, ln, t, f, rg, n)
        for name in ("cu_q", "kv_lens", "taken", "positions", "slots"):
            assert np.array_equal(host(getattr(got, name)), want[name]), name
        assert np.array_equal(host(t), want["table"])
        assert np.array_equal(host(f), free) and np.array_equal(host(rg), ring) and np.array_equal(host(ln), old)


def test_plan_into_given_buffers(ops):
    pool = ops.PagePool(40, 3, 6)
    new = dev([5, 70, 0])
    a = pool.plan(new, 80)
    b = ops.PagePlan(*(torch.full_like(x, 99) for x in a))
    assert pool.plan(new, 80, out=b) is b
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("num", [30, 14])
def test_pool_serves_requests_to_the_end(ops, num):
    """Requests come, grow and finish: no page is lost, doubled or shared, and every slot of a request keeps its page."""
    r = np.random.RandomState(0)
    B, W = 9, 7
    pool = ops.PagePool(num, B, W)
    lengths = np.zeros(B, np.int64)
    table = host(pool.table).copy()
    free, ring = host(pool.free).copy(), host(pool.ring).copy()
    refused = 0
    for step in range(60):
        new = np.where(r.rand(B) < 0.7, np.where(lengths == 0, r.randint(1, 200, B), r.randint(0, 3, B)), 0)
        n = int(new.sum())
        want = oracle.plan(new, lengths, table, free, ring, n)
        plan = pool.plan(dev(new), n)
        assert np.array_equal(host(plan.slots), want["slots"]) and np.array_equal(host(plan.taken), want["taken"])
        ok = want["taken"] >= 0
        refused += int((~ok).sum())
        finished = (r.rand(B) < 0.15) | (lengths + new > 300)
        pool.commit(plan, torch.as_tensor(finished).cuda())
        # the same by hand
        table = want["table"]
        ring[0] = (ring[0] + want["taken"][ok].sum()) % num
        ring[1] -= want["taken"][ok].sum()
        lengths = np.where(ok, want["kv_lens"], lengths)
        for b in np.flatnonzero(finished):
            for j in range(-(-lengths[b] // PAGE)):
                free[(ring[0] + ring[1]) % num] = table[b, j]
                ring[1] += 1
            lengths[b] = 0
        assert np.array_equal(host(pool.lengths), lengths) and np.array_equal(host(pool.ring), ring)
        assert np.array_equal(host(pool.free)[(ring[0] + np.arange(ring[1])) % num], free[(ring[0] + np.arange(ring[1])) % num])
        held = [table[b, j] for b in range(B) for j in range(-(-lengths[b] // PAGE))]
        left = free[(ring[0] + np.arange(ring[1])) % num].tolist()
        assert sorted(held + left) == list(range(num))
    assert num > 14 or refused > 0                      # the small pool runs out at times


def test_commit_twice_takes_once(ops):
    pool = ops.PagePool(10, 2, 4)
    plan = pool.plan(dev([100, 3]), 103)
    pool.commit(plan)
    pool.commit(plan)
    assert host(pool.lengths).tolist() == [100, 3] and host(pool.ring).tolist() == [3, 7]


# ----------------------------------------------------------------- append --
def layout(old, new, seed, spare=2, pad=0):
    """positions, slots (padding: -1), a table and the pages of a pool that holds the step."""
    r = np.random.RandomState(seed)
    old, new = np.asarray(old), np.asarray(new)
    have = -(-(old + new) // PAGE)
    total = int(have.sum()) + spare
    ids = r.permutation(total)
    table = np.full((len(old), max(1, int(have.max()))), -1)
    at = 0
    for b, h in enumerate(have):
        table[b, :h] = ids[at:at + h]
        at += h
    pos = np.concatenate([old[b] + np.arange(new[b]) for b in range(len(old))] + [np.zeros(pad, int)]).astype(int)
    rows = np.concatenate([np.full(new[b], b) for b in range(len(old))] + [np.full(pad, -1)]).astype(int)
    slots = np.array([table[b, p // PAGE] * PAGE + p % PAGE if b >= 0 else -1 for b, p in zip(rows, pos)])
    return pos, slots.astype(int), table, total


def filled_cache(ops, pages, hkv, d, seed, garbage=True):
    """Random codes (every byte, NaN too, where garbage) and scales."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = ops.paged_kv_cache(pages, hkv, d)
    for t in (c.k, c.v):
        b = torch.randint(0, 256, t.shape, generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
        if not garbage:
            b = torch.where((b & 0x7f) == 0x7f, b ^ 1, b)
        t.view(torch.uint8).copy_(b)
    for s in (c.k_scale, c.v_scale):
        s.copy_(2.0 ** torch.randint(-9, -4, s.shape, generator=g, device="cuda").float())
    return c


def to_host(c):
    return type(c)(*(t.cpu() for t in c))


APPENDS = {
    # old, new, hq, hkv, d, far (added to the rotation's positions), padding rows
    "one token": ([0], [1], 4, 2, 128, 0, 0),
    "decode": ([5, 63, 64, 127, 1000], [1] * 5, 8, 2, 128, 0, 0),
    "prompt": ([0], [200], 4, 4, 128, 0, 0),
    "continued": ([10, 64, 3], [150, 64, 61], 4, 1, 128, 0, 3),
    "narrow": ([10, 0, 7], [150, 1, 2], 12, 2, 64, 0, 1),
    "far positions": ([0, 60], [3, 70], 2, 2, 128, 1 << 20, 0),
    "one head each": ([1], [5], 1, 1, 64, 0, 0),
    "many heads": ([1, 2], [5, 1], 40, 8, 128, 0, 0),
    "long batch": ([0, 70], [1500, 3], 4, 2, 128, 0, 5),
    "prompts beside many": ([5, 63, 64, 100] * 80 + [0, 20], [1] * 320 + [700, 90], 2, 1, 64, 0, 3),
    "a few each of many": ([5, 63, 0, 50, 16] * 60, [3, 16, 40, 14, 17] * 60, 2, 2, 128, 0, 0),
    "one kv head, more tokens than a window": ([18, 50, 62] * 150, [1] * 450, 2, 1, 64, 0, 1),
    "longer batch": ([0, 30, 64], [4200, 900, 1], 2, 1, 64, 0, 2),
}


def check_append(ops, old, new, hq, hkv, d, far=0, pad=0, seed=0, mend=None, stride=0):
    pos, slots, _, pages = layout(old, new, seed, pad=pad)
    pos = pos + far
    N = len(pos)
    g = torch.Generator()
    g.manual_seed(seed)
    width = (hq + 2 * hkv) * d
    qkv = (torch.randn(N, width + stride, generator=g) * (0.3 + 2 * torch.rand(width + stride, generator=g))).to(torch.bfloat16)
    if mend:
        mend(qkv)
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=g)).to(torch.bfloat16) for _ in range(2))
    cache = filled_cache(ops, pages, hkv, d, seed)
    before = to_host(type(cache)(*(t.clone() for t in cache)))
    q_out = torch.full((N, hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_qk_norm_rope_kv(qkv.cuda()[:, :width], qw.cuda(), kw.cuda(), dev(pos), dev(slots), ops.rope_turns(THETA, d),
                              cache, q_out, hq, hkv, d, EPS)
    after = to_host(cache)

    x = qkv[:, :width].double().view(N, hq + 2 * hkv, d)
    # fp32 against 64 bits: the mean of D squares, its root, two products and the turn each lose a few 2^-24 of the
    # pair's size; the angle is off by 2^-25 turns + 2^-65 * position, 2^-22.3 radians: 2^-19 of the pair in all
    q, size = oracle.norm_rope(x[:, :hq], qw.double(), pos, THETA, EPS)
    assert torch.all((q_out.cpu().double() - q).abs() <= q.abs() * 2.0 ** -8 + size * 2.0 ** -18) or bool(mend)
    k, size = oracle.norm_rope(x[:, hq:hq + hkv], kw.double(), pos, THETA, EPS)
    v = x[:, hq + hkv:]
    check_pages(before, after, k, v, size, slots, hkv)
    return q_out, after


def check_pages(before, after, k, v, size, slots, hkv):
    bad = ~(k.isfinite().all(-1) & v.isfinite().all(-1))
    touched = {}
    for i, s in enumerate(slots):
        if s >= 0:
            touched.setdefault(int(s) // PAGE, []).append(i)
    for page in range(before.k.shape[0]):
        toks = touched.get(page, [])
        offs = [int(slots[i]) % PAGE for i in toks]
        for h in range(hkv):
            for name, val, slack in (("k", k, size), ("v", v, None)):
                codes_b, codes_a = getattr(before, name)[page, h], getattr(after, name)[page, h]
                s_b, s_a = (float(getattr(c, name + "_scale")[page, h]) for c in (before, after))
                if name == "v":
                    codes_b, codes_a = codes_b.view(torch.uint8).T.view(torch.float8_e4m3fn), codes_a.view(torch.uint8).T.view(torch.float8_e4m3fn)
                if not toks:
                    assert torch.equal(codes_b.view(torch.uint8), codes_a.view(torch.uint8)) and s_a == s_b
                    continue
                good = [i for i in toks if not bad[i, h]]
                amax = max([float(val[i, h].abs().max()) for i in good], default=0.0)
                err = max([float(slack[i, h].max()) for i in good], default=0.0) * 2.0 ** -18 if slack is not None else 0.0
                lo, hi = (oracle.scale_for(max(0.0, amax + e)) for e in (-err, err))
                if min(offs) > 0:
                    lo, hi = max(lo, s_b), max(hi, s_b)
                assert lo <= s_a <= hi, (name, page, h, lo, s_a, hi)
                # older tokens: their codes times the change of scale, rounded once more (exactly as a cast does)
                first = min(offs)
                old = (codes_b[:first].float() * (s_b / s_a)).to(torch.float8_e4m3fn)
                assert torch.equal(old.float().nan_to_num(1e9), codes_a[:first].float().nan_to_num(1e9))
                # slots that no token of the step has
                rest = [o for o in range(first, PAGE) if o not in offs]
                assert torch.equal(codes_b.view(torch.uint8)[rest], codes_a.view(torch.uint8)[rest])
                for i, o in zip(toks, offs):
                    got = codes_a[o].float().double() * s_a
                    if bad[i, h]:
                        assert got.isnan().all() if name == "k" else (got == 0).all()
                        continue
                    ref = val[i, h]
                    # half a step: 2^-4 of the value, or half of the smallest code's 2^-9; a value past 448 is cut to it
                    tol = ref.abs() * 2.0 ** -4 + 2.0 ** -10 * s_a + err
                    assert torch.all((got - ref.clamp(-448 * s_a, 448 * s_a)).abs() <= tol), (name, page, h, o)


@pytest.mark.parametrize("case", APPENDS, ids=list(APPENDS))
def test_append(ops, case):
    check_append(ops, *APPENDS[case])


def test_append_strided_rows(ops):
    check_append(ops, [3, 0], [70, 2], 4, 2, 128, stride=24)


def test_append_raises_and_keeps_scales(ops):
    """Tokens behind others: larger ones raise the page's scale, smaller ones leave it."""
    for factor in (2.0 ** 9, 2.0 ** -9, 2.0 ** 40):
        def mend(x, f=factor):
            x *= f
        check_append(ops, [7, 100], [3, 1], 4, 2, 128, mend=mend)


def test_append_zeros(ops):
    def mend(x):
        x.zero_()
    q, after = check_append(ops, [0, 3], [10, 4], 4, 2, 128, mend=mend)
    assert (q.cpu() == 0).all()


def test_append_not_finite(ops):
    def mend(x):
        d, hq, hkv = 128, 4, 2
        x[2, (hq + 0) * d + 5] = math.nan             # K of head 0
        x[3, (hq + hkv + 1) * d + 9] = math.inf       # V of head 1
        x[70, (hq + 1) * d + 127] = -math.inf         # K of head 1
    check_append(ops, [0], [80], 4, 2, 128, mend=mend)


def test_append_huge_values(ops):
    def mend(x):
        x[:, 6 * 128:] = 3.3e38                       # V: past 448 * 2^119, cut to it
        x[1, 6 * 128:] = -1e-38
    check_append(ops, [0], [5], 4, 2, 128, mend=mend)


@pytest.mark.parametrize("hkv,d,seed", [(1, 64, 0), (1, 128, 1), (3, 64, 2), (8, 128, 3)])
def test_append_in_one_call_or_many(ops, hkv, d, seed):
    """Every bit is the same, however the requests are dealt out: prompts, chunks, a few tokens each and single ones."""
    r = np.random.RandomState(seed)
    new = r.choice([0, 1, 1, 2, 5, 16, 33, 70], 250)
    new[r.randint(250)] = 1500
    pos, slots, _, pages = layout(r.randint(0, 300, 250), new, seed)
    hq, n, start = 2 * hkv, int(new.sum()), np.concatenate([[0], np.cumsum(new)])
    qkv = torch.randn(n, (hq + 2 * hkv) * d, device="cuda").to(torch.bfloat16) * 2
    w, turns = torch.ones(d, dtype=torch.bfloat16, device="cuda"), ops.rope_turns(THETA, d)
    got = []
    for cuts in ([0, 250], range(0, 251, 10)):
        cache, q = filled_cache(ops, pages, hkv, d, seed), torch.zeros(n, hq, d, dtype=torch.bfloat16, device="cuda")
        for a, b in zip(cuts, list(cuts)[1:]):
            i, j = start[a], start[b]
            ops.paged_qk_norm_rope_kv(qkv[i:j], w, w, dev(pos[i:j]), dev(slots[i:j]), turns, cache, q[i:j], hq, hkv, d, EPS)
        got.append([t.view(torch.uint8) for t in (*cache, q)])
    assert all(torch.equal(x, y) for x, y in zip(*got))


def test_append_slots_outside_the_cache(ops):
    """Rows whose slot is negative or past the last page append nothing; q is written for all."""
    cache = filled_cache(ops, 3, 2, 128, 1)
    before = [t.clone() for t in cache]
    q_out = torch.zeros(4, 4, 128, dtype=torch.bfloat16, device="cuda")
    qkv = torch.randn(4, 8 * 128, device="cuda").to(torch.bfloat16)
    w = torch.ones(128, device="cuda", dtype=torch.bfloat16)
    ops.paged_qk_norm_rope_kv(qkv, w, w, dev([0, 1, 2, 3]), dev([-1, 192, 2**31 - 1, -(2**31)]), ops.rope_turns(THETA, 128),
                              cache, q_out, 4, 2, 128, EPS)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, cache))
    assert (q_out != 0).any(-1).all()


def test_append_nothing(ops):
    cache = ops.paged_kv_cache(1, 1, 64)
    e = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
    ops.paged_qk_norm_rope_kv(e(0, 192), e(64), e(64), e(0, dt=torch.int32), e(0, dt=torch.int32), ops.rope_turns(THETA, 64),
                              cache, e(0, 1, 64), 1, 1, 64, EPS)


# -------------------------------------------------------------- attention --
ATTNS = {
    # old, new, hq, hkv, d
    "one key": ([0], [1], 4, 1, 128),
    "single": ([8190], [1], 32, 8, 128),
    "decode": ([0, 62, 63, 64, 200, 1], [1] * 6, 8, 2, 128),
    "groups of one": ([100, 5], [1, 1], 4, 4, 64),
    "group of five": ([130, 70], [1, 3], 10, 2, 128),
    "group of sixteen": ([300], [1], 32, 2, 64),
    "group of forty": ([70, 3], [2, 1], 40, 1, 64),
    "a few each": ([100, 0, 64, 63], [5, 4, 2, 3], 8, 2, 128),
    "rows of a tile's end": ([100, 30], [4, 8], 8, 2, 128),
    "prompt": ([0], [300], 8, 2, 128),
    "prompts": ([0, 0, 64], [65, 128, 191], 4, 4, 64),
    "chunk beside decode": ([500, 77, 0, 200], [130, 1, 40, 1], 8, 2, 128),
    "chunk beside decode, heads of 64": ([700, 77, 0, 200], [300, 1, 40, 1], 4, 4, 64),
    "prompts, heads of 64": ([0, 0, 64], [65, 328, 391], 4, 4, 64),
    "chunk beside a few, heads of 64": ([700, 77, 0, 200, 30], [600, 1, 40, 17, 16], 8, 4, 64),
    "a few each of many": ([200] * 30, [33, 8, 9, 16, 64] * 6, 16, 2, 128),
    "few rows": ([300, 10], [100, 27], 8, 2, 128),
    "rows without tokens": ([10, 50, 0], [0, 2, 0], 4, 2, 128),
    "ragged decode": ([3000, 1, 70, 900, 0, 511, 64, 2100], [1] * 8, 16, 2, 128),
    "long chunk": ([700], [600], 4, 1, 128),
    "wide rows": ([90], [100], 6, 2, 64),
}


def attention_case(ops, old, new, hq, hkv, d, seed=0, pad=3):
    pos, slots, table, pages = layout(old, new, seed)
    N = len(pos)
    # garbage in every slot that no request has: NaN codes too.  Live slots hold finite codes
    cache = filled_cache(ops, pages, hkv, d, seed)
    live = torch.zeros(pages, PAGE, dtype=torch.bool)
    for b in range(len(old)):
        for p in range(old[b] + new[b]):
            live[table[b, p // PAGE], p % PAGE] = True
    for t, m in ((cache.k, live[:, None, :, None]), (cache.v, live[:, None, None, :])):
        b = t.view(torch.uint8)
        b.copy_(torch.where(m.cuda() & ((b & 0x7f) == 0x7f), b ^ 1, b))
    # codes reach 448: with scales of 2^-9 .. 2^-5 keys of size 1 to 14, so that the softmax is peaked in places
    g = torch.Generator()
    g.manual_seed(seed + 1)
    q = (torch.randn(N + pad, hq, d, generator=g) * 0.3).to(torch.bfloat16)
    cu = np.concatenate([[0], np.cumsum(new)])
    return q, cache, table, cu, np.asarray(old) + np.asarray(new)


def check_attention(ops, q, cache, table, cu, kv_lens, hq, hkv, d, scale=None, **kw):
    scale = scale or 1 / math.sqrt(d)
    out = torch.full((q.shape[0], hq * d), 5.0, dtype=torch.bfloat16, device="cuda")
    got = ops.paged_attention(q.cuda(), cache, dev(table), dev(cu), dev(kv_lens), hq, hkv, d, scale, out=out, **kw)
    assert got is out
    hc = to_host(cache)
    hc.k.view(torch.uint8).copy_(torch.where((hc.k.view(torch.uint8) & 0x7f) == 0x7f, 0, hc.k.view(torch.uint8)))
    hc.v.view(torch.uint8).copy_(torch.where((hc.v.view(torch.uint8) & 0x7f) == 0x7f, 0, hc.v.view(torch.uint8)))
    o, size = oracle.attention(q, hc, table, cu, kv_lens, hq, hkv, scale)
    o, size = (x.reshape(len(q), -1) for x in (o, size))
    end = int(cu[-1])
    # each weight is rounded to bf16 (2^-8), the output too; scores in fp32: |q|.|k| scale is below 2^9 here and its D
    # products and sums lose under 2^-19 of it, 2^-10 of a weight
    tol = size * (2.0 ** -8 + 2.0 ** -9) + o.abs() * 2.0 ** -8 + 2.0 ** -100
    diff = (out[:end].cpu().double() - o[:end]).abs()
    assert torch.all(diff <= tol[:end]), float((diff / tol[:end]).max())
    assert (out[end:] == 5.0).all()                   # rows behind the last request
    return out


@pytest.mark.parametrize("case", ATTNS, ids=list(ATTNS))
def test_attention(ops, case):
    old, new, hq, hkv, d = ATTNS[case]
    args = attention_case(ops, old, new, hq, hkv, d)
    a = check_attention(ops, *args, hq, hkv, d)
    work = ops.paged_attention_workspace(len(args[0]), len(old), hq, hkv, d)
    b = check_attention(ops, *args, hq, hkv, d, max_new=max(new), work=work)
    c = check_attention(ops, *args, hq, hkv, d, max_new=max(new), work=work)
    assert torch.equal(b, c)                          # the same bits again
    assert a.shape == b.shape


@pytest.mark.parametrize("rows,long,seed", [(65, 0, 0), (130, 150, 1), (200, 0, 2), (1024, 100, 3)])
def test_attention_many_requests(ops, rows, long, seed):
    """More requests than a wave has lanes, some without tokens, with and without a chunk among them."""
    r = np.random.RandomState(seed)
    old, new = r.randint(0, 150, rows), r.randint(0, 3, rows)
    old[r.randint(rows)] = 900
    if long:
        new[r.randint(rows)] = long
    q, cache, table, cu, kv = attention_case(ops, old, new, 4, 2, 64, seed)
    check_attention(ops, q, cache, table, cu, kv, 4, 2, 64)


def test_attention_rows_that_see_nothing(ops):
    """A request that was not admitted (no keys), and one with fewer keys than rows: zeros where no key is seen."""
    q, cache, table, cu, kv = attention_case(ops, [10, 0, 20], [3, 5, 2], 4, 2, 128)
    kv = np.array([13, 3, 0])
    out = check_attention(ops, q, cache, table, cu, kv, 4, 2, 128)
    assert (out[3:5] == 0).all() and (out[8:10] == 0).all() and (out[5:8] != 0).any()


@pytest.mark.parametrize("new", [1, 50, 200])
def test_attention_bad_pages(ops, new):
    """A page that the cache does not have counts as masked; a row left with none gives zeros."""
    q, cache, table, cu, kv = attention_case(ops, [200, 300, 20], [new] * 3, 4, 2, 128)
    table[0, 1], table[1, 0], table[1, 3] = -1, cache.k.shape[0], 2**31 - 1
    table[2, :] = -5
    out = check_attention(ops, q, cache, table, cu, kv, 4, 2, 128)
    assert (out[2 * new:3 * new] == 0).all()


@pytest.mark.parametrize("new", [1, 50, 200])
def test_attention_bad_pages_beside_an_unwritten_first_page(ops, new):
    """The cache's first page, never written: scales and codes of any bits.  Masked pages take nothing from it."""
    q, cache, table, cu, kv = attention_case(ops, [200, 300, 20], [new] * 3, 4, 2, 128)
    first = lambda t, v: torch.cat([torch.full_like(t[:1].view(torch.uint8), v), t.view(torch.uint8)]).view(t.dtype)  # noqa: E731
    cache = ops.PagedKV(*(first(t, 0xff) for t in cache))      # NaN codes and NaN scales
    table = table + 1
    table[0, 1], table[1, 0], table[1, 3] = -1, cache.k.shape[0], 2**31 - 1
    table[2, :] = -5
    out = ops.paged_attention(q.cuda(), cache, dev(table), dev(cu), dev(kv), 4, 2, 128, 0.1)
    assert out[:3 * new].isfinite().all() and (out[2 * new:3 * new] == 0).all()
    for t in cache:
        t[0].view(torch.uint8).zero_()
    assert torch.equal(out, ops.paged_attention(q.cuda(), cache, dev(table), dev(cu), dev(kv), 4, 2, 128, 0.1))


def test_attention_shared_pages(ops):
    """Two requests with the same prefix read the same pages."""
    q, cache, table, cu, kv = attention_case(ops, [128, 128], [1, 1], 4, 2, 128)
    table[1, :2] = table[0, :2]
    check_attention(ops, q, cache, table, cu, kv, 4, 2, 128)


@pytest.mark.parametrize("new", [1, 40, 200])
def test_attention_nan_key(ops, new):
    """A NaN key reaches exactly the rows that see it, in its head."""
    q, cache, table, cu, kv = attention_case(ops, [70, 70], [new, new], 4, 2, 128)
    at = 70 + new // 2 if new > 1 else 3              # a position in the chunk, or an old one
    cache.k.view(torch.uint8)[table[0, at // PAGE], 1, at % PAGE, 17] = 0x7f
    out = ops.paged_attention(q.cuda(), cache, dev(table), dev(cu), dev(kv), 4, 2, 128, 0.1).view(-1, 4, 128)
    sees = torch.arange(new) + 70 >= at
    assert out[:new, 2:][sees.cuda()].isnan().all()
    rest = out.clone()
    rest[:new, 2:][sees.cuda()] = 0
    assert rest[:2 * new].isfinite().all()


def test_attention_large_scores(ops):
    """Scores far apart: the maximum moves along the pages and nothing overflows."""
    q, cache, table, cu, kv = attention_case(ops, [300, 5], [1, 90], 4, 2, 128)
    big = ops.PagedKV(cache.k, cache.v, cache.k_scale * 16, cache.v_scale)
    # the scores reach thousands: fp32 keeps them to 2^-11, so compare with the oracle at the sizes of the values only
    out = ops.paged_attention(q.cuda(), big, dev(table), dev(cu), dev(kv), 4, 2, 128, 1.0)
    assert out[:91].isfinite().all()


def test_attention_equal_scores(ops):
    """q = 0: the mean of V, whatever the order of the pages."""
    q, cache, table, cu, kv = attention_case(ops, [1000, 64], [1, 7], 4, 2, 128)
    check_attention(ops, q * 0, cache, table, cu, kv, 4, 2, 128)


def test_attention_workspace_too_small(ops):
    """Room for few rows does not do for many; nothing is launched."""
    q, cache, table, cu, kv = attention_case(ops, [0], [300], 4, 2, 128)
    few = ops.paged_attention_workspace(1, 1, 4, 2, 128)
    for work in (few, few[:100]):
        with pytest.raises(ValueError, match="workspace"):
            ops.paged_attention(q.cuda(), cache, dev(table), dev(cu), dev(kv), 4, 2, 128, 0.1, work=work)
    for bad in (few.double(), few[::2], few[1:], few.view(1, -1), few.cpu()):
        with pytest.raises(ValueError, match="paged_attention"):
            ops.paged_attention(q.cuda(), cache, dev(table), dev(cu), dev(kv), 4, 2, 128, 0.1, work=bad)


def test_attention_one_workspace_for_all(ops):
    """Steps of other sizes, heads and kinds in turn on one workspace: each finds it as the first did."""
    work = ops.paged_attention_workspace(1024, 64, 32, 1, 128)
    for name in list(ATTNS) + ["single", "chunk beside decode", "prompts", "group of sixteen"]:
        old, new, hq, hkv, d = ATTNS[name]
        q, cache, table, cu, kv = attention_case(ops, old, new, hq, hkv, d)
        check_attention(ops, q, cache, table, cu, kv, hq, hkv, d, work=work)
    assert (work[:1024] == 0).all()


def test_attention_more_new_tokens_than_said(ops):
    q, cache, table, cu, kv = attention_case(ops, [500, 77, 0], [130, 1, 70], 8, 2, 128)
    for said in (0, 1, 16, 17, 130):
        check_attention(ops, q, cache, table, cu, kv, 8, 2, 128, max_new=said)


@pytest.mark.parametrize("new", [3, 90, 300])
def test_attention_overlapping_requests_stay_in_bounds(ops, new):
    """Rows that several requests claim have no answer, but nothing outside them is touched and the next call is right."""
    q, cache, table, cu, kv = attention_case(ops, [2000] * 6, [new] * 6, 4, 2, 128)
    work = ops.paged_attention_workspace(6 * new, 6, 4, 2, 128)
    out = torch.full((6 * new + 3, 512), 5.0, dtype=torch.bfloat16, device="cuda")
    n = 6 * new
    ops.paged_attention(q.cuda(), cache, dev(table), dev([0, n, 0, n, 0, n, n]), dev(kv), 4, 2, 128, 0.1, out=out, work=work)
    assert (out[n:] == 5.0).all()
    check_attention(ops, q, cache, table, cu, kv, 4, 2, 128, work=work)


@pytest.mark.parametrize("name", ["single", "long chunk", "chunk beside decode"])
def test_attention_same_bits(ops, name):
    """Whichever part of a tile comes last, a call's result is the same."""
    old, new, hq, hkv, d = ATTNS[name]
    q, cache, table, cu, kv = attention_case(ops, old, new, hq, hkv, d)
    args = (q.cuda(), cache, dev(table), dev(cu), dev(kv), hq, hkv, d, 0.1)
    work = ops.paged_attention_workspace(len(q), len(kv), hq, hkv, d)
    want = ops.paged_attention(*args)
    for _ in range(20):
        assert torch.equal(ops.paged_attention(*args, work=work), want)


def test_attention_nothing(ops):
    cache = ops.paged_kv_cache(1, 1, 64)
    out = ops.paged_attention(torch.empty(0, 1, 64, dtype=torch.bfloat16, device="cuda"), cache, dev([[0]]), dev([0, 0]),
                              dev([0]), 1, 1, 64, 1.0)
    assert out.shape == (0, 64)


def test_attention_long_cache_offsets(ops):
    """Pages whose bytes lie past 2^31 and 2^32 in the cache: 8 heads of 128, 8 KB a page and head and side."""
    pages, hkv, d = 70000, 8, 128                     # 4.6 GB each of K and V
    cache = ops.paged_kv_cache(pages, hkv, d)
    used = [69999, 0, 33000, 66000]
    ids = torch.tensor(used, device="cuda")
    for t in (cache.k, cache.v):
        b = torch.randint(0, 256, (4, *t.shape[1:]), device="cuda", dtype=torch.int32).to(torch.uint8)
        t.view(torch.uint8)[ids] = torch.where((b & 0x7f) == 0x7f, b ^ 1, b)
    cache.k_scale[ids], cache.v_scale[ids] = 2.0 ** -6, 2.0 ** -7
    q = (torch.randn(40, 16, d) * 0.3).to(torch.bfloat16)
    small = ops.PagedKV(*(t.view(torch.uint8)[ids].view(t.dtype) if t.dtype == torch.float8_e4m3fn else t[ids] for t in cache))
    for n in (1, 40):
        args = (q[:n].cuda().contiguous(),)
        a = ops.paged_attention(*args, cache, dev([used]), dev([0, n]), dev([250]), 16, hkv, d, 0.1, max_new=n)
        b = ops.paged_attention(*args, small, dev([[0, 1, 2, 3]]), dev([0, n]), dev([250]), 16, hkv, d, 0.1, max_new=n)
        assert torch.equal(a, b)
    # the append there, against the same append at the front
    w = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    qkv = torch.randn(2, (16 + 2 * hkv) * d, device="cuda").to(torch.bfloat16)
    qo = torch.empty(2, 16, d, dtype=torch.bfloat16, device="cuda")
    for c, page in ((cache, 69999), (small, 0)):
        ops.paged_qk_norm_rope_kv(qkv, w, w, dev([250, 251]), dev([page * 64 + 58, page * 64 + 59]), ops.rope_turns(THETA, d), c,
                                  qo, 16, hkv, d, EPS)
    for x, y in zip(cache, small):
        assert torch.equal(x[69999].view(torch.uint8), y[0].view(torch.uint8))


# --------------------------------------------------------------- together --
def serve_step(ops, s, new, n):
    """One step of a two-layer server on random activations: everything between the matrix products."""
    plan = s["pool"].plan(new, n, out=s["plan"])
    x = s["x"]
    for layer in range(2):
        qkv = torch.matmul(x, s["wqkv"][layer])
        ops.paged_qk_norm_rope_kv(qkv, s["qw"], s["kw"], plan.positions, plan.slots, s["turns"], s["cache"][layer], s["q"],
                                  s["hq"], s["hkv"], s["d"], EPS)
        att = ops.paged_attention(s["q"], s["cache"][layer], s["pool"].table, plan.cu_q, plan.kv_lens, s["hq"], s["hkv"],
                                  s["d"], 1 / math.sqrt(s["d"]), out=s["att"][layer], work=s["work"])
        x = x + torch.matmul(att, s["wo"][layer])
    logits = torch.matmul(x, s["lm"])
    ops.sample(logits, s["u"], s["t"], s["k"], s["p"], s["mp"], tokens=s["tokens"], probs=s["probs"], work=s["swork"])
    s["pool"].commit(plan, s["finished"])
    return plan


def server(ops, n, rows, pages=40, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    hq, hkv, d, hidden, vocab = 8, 2, 128, 256, 1000
    rnd = lambda *sh: (torch.randn(*sh, generator=g, device="cuda") * sh[0] ** -0.5).to(torch.bfloat16)  # noqa: E731
    f = lambda v, dt: torch.full((n,), v, dtype=dt, device="cuda")  # noqa: E731
    pool = ops.PagePool(pages, rows, 8)
    i = dict(dtype=torch.int32, device="cuda")
    return dict(hq=hq, hkv=hkv, d=d, pool=pool, plan=ops.PagePlan(torch.zeros(rows + 1, **i), *(torch.zeros(rows, **i) for _ in range(2)),
                                                                  *(torch.zeros(n, **i) for _ in range(2))),
                x=rnd(n, hidden) * 16, wqkv=[rnd(hidden, (hq + 2 * hkv) * d) for _ in range(2)],
                wo=[rnd(hq * d, hidden) for _ in range(2)], lm=rnd(hidden, vocab),
                qw=torch.ones(d, dtype=torch.bfloat16, device="cuda"), kw=torch.ones(d, dtype=torch.bfloat16, device="cuda"),
                turns=ops.rope_turns(THETA, d), cache=[filled_cache(ops, pages, hkv, d, seed) for _ in range(2)],
                q=torch.zeros(n, hq, d, dtype=torch.bfloat16, device="cuda"),
                att=[torch.zeros(n, hq * d, dtype=torch.bfloat16, device="cuda") for _ in range(2)],
                work=ops.paged_attention_workspace(n, rows, hq, hkv, d), swork=ops.sample_workspace(n, vocab),
                u=torch.rand(n, generator=g, device="cuda"), t=f(0.8, torch.float32), k=f(50, torch.int32), p=f(0.95, torch.float32),
                mp=f(0.01, torch.float32), tokens=torch.zeros(n, dtype=torch.int64, device="cuda"),
                probs=torch.zeros(n, device="cuda"), finished=torch.zeros(rows, dtype=torch.bool, device="cuda"))


def test_steps_together(ops):
    """Prompts, then decode beside a new prompt: each layer's attention is the oracle's over what the pages hold."""
    s = server(ops, 200, 3)
    for new in ([70, 0, 30], [1, 100, 1], [1, 1, 1], [0, 1, 66]):
        before = host(s["pool"].lengths).copy()
        s["x"].add_(0.125)                            # other tokens
        plan = serve_step(ops, s, dev(new), 200)
        n = sum(new)
        assert np.array_equal(host(s["pool"].lengths), before + new)
        for layer in range(2):
            if layer == 1:                            # s["q"] holds the last layer's
                c = to_host(s["cache"][layer])
                for t in (c.k, c.v):
                    t.view(torch.uint8).copy_(torch.where((t.view(torch.uint8) & 0x7f) == 0x7f, 0, t.view(torch.uint8)))
                o, size = oracle.attention(s["q"].cpu(), c, host(s["pool"].table), host(plan.cu_q), host(plan.kv_lens), 8, 2, 1 / math.sqrt(128))
                o, size = o.reshape(200, -1), size.reshape(200, -1)
                tol = size * (2.0 ** -8 + 2.0 ** -9) + o.abs() * 2.0 ** -8 + 2.0 ** -100
                assert torch.all((s["att"][layer].cpu().double() - o).abs()[:n] <= tol[:n])
        assert (host(s["tokens"])[:n] >= 0).all() and (host(s["tokens"])[:n] < 1000).all()


def test_captured_step_replays(ops):
    """A captured decode step against the same steps run eagerly, with eager work and synchronisations in between."""
    a, b = server(ops, 4, 4, seed=3), server(ops, 4, 4, seed=3)
    new = dev([1, 1, 0, 1])
    for s in (a, b):                                  # also the warm-up of the library's products
        for _ in range(3):
            serve_step(ops, s, new, 4)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        serve_step(ops, a, new, 4)
    for step in range(70):                            # over a page border
        for s in (a, b):
            s["x"].add_(0.0625)
        g.replay()
        if step % 7 == 3:
            torch.cuda.synchronize()
        serve_step(ops, b, new, 4)
        if step % 5 == 0:
            assert torch.equal(a["tokens"], b["tokens"]) and torch.equal(a["att"][1][:3], b["att"][1][:3])
            assert torch.equal(a["probs"], b["probs"])
    assert torch.equal(a["pool"].lengths, b["pool"].lengths) and host(a["pool"].lengths).tolist() == [73, 73, 0, 73]
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for p, q in zip(a["cache"], b["cache"]) for x, y in zip(p, q))


def test_two_streams(ops):
    """Calls on two streams at once, each with buffers of its own, give what they give alone."""
    servers = [server(ops, 64, 4, seed=i) for i in (1, 2)]
    new = dev([16, 16, 16, 16])
    want = []
    for i in (1, 2):
        s = server(ops, 64, 4, seed=i)
        for _ in range(5):
            serve_step(ops, s, new, 64)
        want.append((s["att"][1].clone(), s["tokens"].clone()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, s in zip(streams, servers):
            with torch.cuda.stream(st):
                serve_step(ops, s, new, 64)
    torch.cuda.synchronize()
    for s, (att, tok) in zip(servers, want):
        assert torch.equal(s["att"][1], att) and torch.equal(s["tokens"], tok)


def test_plan_of_as_many_rows_as_there_are_indices(ops):
    """2^31 - 1 rows of which 75 hold a token: the walk over them ends at the last one."""
    pool, n = ops.PagePool(40, 3, 6), 2**31 - 1
    small, plan = pool.plan(dev([5, 70, 0]), 75), pool.plan(dev([5, 70, 0]), n)
    assert plan.slots.shape == (n,) and plan.cu_q.tolist() == [0, 5, 75, 75] and plan.taken.tolist() == [1, 2, 0]
    assert torch.equal(plan.slots[:75], small.slots) and torch.equal(plan.positions[:75], small.positions)
    for t, v in ((plan.slots, -1), (plan.positions, 0)):
        assert int(t[75:].amin()) == v and int(t[75:].amax()) == v


@pytest.mark.parametrize("new", [1, 50, 300])
def test_attention_scales_that_are_no_powers_of_two(ops, new):
    """Rows that see a page with such a scale (of K or of V, in their head) give NaN, all others what they give without."""
    q, cache, table, cu, kv = attention_case(ops, [200, 300, 20], [new] * 3, 4, 2, 128)
    args = (dev(table), dev(cu), dev(kv), 4, 2, 128, 0.1)
    want = ops.paged_attention(q.cuda(), cache, *args)
    last = (20 + new - 1) // PAGE                             # the third request's page that only its last rows see
    above_one = float(np.nextafter(np.float32(1), np.float32(2)))
    for bad in (1.5 * 2.0 ** -7, 1 / 448, above_one, -(2.0 ** -6), 0.0, math.inf, math.nan, 2.0 ** -111, 2.0 ** 120, 2.0 ** -149):
        for side, b, h, page in (("k_scale", 0, 1, 1), ("v_scale", 1, 0, 0), ("v_scale", 2, 1, last)):
            scale = getattr(cache, side).clone()
            scale[table[b, page], h] = bad
            got = ops.paged_attention(q.cuda(), cache._replace(**{side: scale}), *args).view(-1, 4, 128)
            lost = torch.zeros(got.shape[:2], dtype=torch.bool)
            lost[b * new:(b + 1) * new, 2 * h:2 * h + 2] = (torch.arange(new) + [200, 300, 20][b] >= page * PAGE)[:, None]
            assert bool(lost.any()) and torch.equal(got.isnan().all(-1).cpu(), lost), (bad, side)
            assert torch.equal(got[~lost.cuda()], want.view(-1, 4, 128)[~lost.cuda()]), (bad, side)
    one = ops.paged_attention(q.cuda(), cache._replace(v_scale=torch.ones_like(cache.v_scale)), *args)
    for e in (-110, 100):
        far = cache._replace(v_scale=torch.full_like(cache.v_scale, 2.0 ** e))
        assert torch.equal(ops.paged_attention(q.cuda(), far, *args), one * 2.0 ** e)


@pytest.mark.parametrize("new,rows,hq,hkv", [(1, 520, 2, 1), (900, 1, 16, 8)])
def test_attention_more_pages_than_lanes(ops, new, rows, hq, hkv):
    """A wave's (a workgroup's) pages come in rounds of 64: requests of 300 shared pages, too many to be split far."""
    r, d, pages = np.random.RandomState(0), 64, 300
    cache = filled_cache(ops, pages, hkv, d, 1, garbage=False)
    table, kv = r.randint(0, pages, (rows, 300)), r.randint(17000, 19201, rows)
    q = (torch.randn(rows * new, hq, d) * 0.3).to(torch.bfloat16)
    some = [0, rows // 3, rows - 1] if rows > 1 else [0]
    for odd in (False, True):
        if odd:                                       # past the first round, of one head
            table[some[-1], 250] = pages
            cache = ops.PagedKV(*(torch.cat([t.view(torch.uint8), t[:1].view(torch.uint8)]).view(t.dtype) for t in cache))
            cache.k_scale[pages, 0] = 0.3
        out = ops.paged_attention(q.cuda(), cache, dev(table), dev(np.arange(rows + 1) * new), dev(kv), hq, hkv, d, 0.125)
        out = out.view(rows, new, hq, d)[some].cpu()
        if odd:
            assert out[-1, :, :hq // hkv].isnan().all()
            assert out[:-1].isfinite().all() and out[:, :, hq // hkv:].isfinite().all()
            continue
        want, size = oracle.attention(q.view(rows, new, hq, d)[some].reshape(-1, hq, d), to_host(cache), table[some],
                                      np.arange(len(some) + 1) * new, kv[some], hq, hkv, 0.125)
        want, size = want.view(out.shape), size.view(out.shape)
        # as in check_attention
        tol = size * (2.0 ** -8 + 2.0 ** -9) + want.abs() * 2.0 ** -8 + 2.0 ** -100
        assert torch.all((out.double() - want).abs() <= tol)


@pytest.mark.parametrize("longs", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_parts_are_resident(ops, d, longs):
    """The parts that a call aims at have a place on the CUs: more would only add to the join."""
    fit = ctypes.c_int(0)
    aim = ops.lib().mivgpu_paged_attention_resident(d, longs, ctypes.byref(fit))
    assert 1 <= aim <= fit.value


def test_attention_as_many_pages_as_there_are_indices(ops):
    """64 tiles of 2^25 - 1 pages, one below 2^31 in all: none but a request's last is in the cache."""
    W, n = 2**25 - 1, 64
    cache = filled_cache(ops, 2, 1, 64, 0, garbage=False)
    q = torch.randn(n, 16, 64, device="cuda").to(torch.bfloat16)
    want = ops.paged_attention(q, cache, dev([[1]]), dev([0, n]), dev([PAGE]), 16, 1, 64, 0.125, max_new=1)   # the same kernel
    table = torch.full((1, W), -1, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    out = torch.full((n, 16 * 64), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention(q, cache, table, dev([0, n]), dev([W * PAGE]), 16, 1, 64, 0.125, max_new=1, out=out)
    assert torch.equal(out, want)


# ------------------------------------------------- closer looks at the same --
@pytest.mark.parametrize("grow", [1, -1])
@pytest.mark.parametrize("case", ["single", "a few each", "prompts", "chunk beside decode", "long chunk", "chunk beside a few, heads of 64"])
def test_attention_scores_that_grow_along_the_pages(ops, case, grow):
    """Keys of twice the size from page to page (or half), queries from 2^-6 to 2^6: maxima that move by less and by more
    than a factor of 2^8 of the weights, scores in the thousands.  A query has one value that is not zero, so that its
    scores are exact in fp32 and the bounds are those of check_attention."""
    old, new, hq, hkv, d = ATTNS[case]
    q, cache, table, cu, kv = attention_case(ops, old, new, hq, hkv, d)
    r = np.random.RandomState(1)
    for b in range(len(kv)):
        for j in range(-(-int(kv[b]) // PAGE)):
            cache.k_scale[table[b, j]] = 2.0 ** (-9 + (j if grow > 0 else -j) % 10)
    one = torch.zeros(q.numel() // d, d, dtype=torch.bfloat16)
    at, size = r.randint(0, d, len(one)), 2.0 ** r.randint(-6, 7, len(one)) * r.choice([-1, 1], len(one))
    one[torch.arange(len(one)), torch.as_tensor(at)] = torch.as_tensor(size).to(torch.bfloat16)
    check_attention(ops, one.view(q.shape), cache, table, cu, kv, hq, hkv, d, scale=1.0)


@pytest.mark.parametrize("old,new,hq,hkv,d", [
    ([500], [2048], 16, 16, 128), ([500], [2048], 32, 8, 128), ([2000], [512], 16, 16, 64), ([0], [1100], 16, 16, 64),
    ([700, 2000, 64, 900], [700, 1, 3, 1], 16, 16, 64), ([0, 300, 4000], [1000, 900, 1], 8, 4, 128)])
def test_attention_tiles_of_unlike_lengths(ops, old, new, hq, hkv, d):
    """Prompts and chunks of some tiles a head, the last of several times the first one's pages, with CUs over."""
    q, cache, table, cu, kv = attention_case(ops, old, new, hq, hkv, d, seed=4)
    work = ops.paged_attention_workspace(len(q), len(old), hq, hkv, d)
    a = check_attention(ops, q, cache, table, cu, kv, hq, hkv, d, work=work)
    for _ in range(3):
        out = torch.full_like(a, 5.0)
        ops.paged_attention(q.cuda(), cache, dev(table), dev(cu), dev(kv), hq, hkv, d, 1 / math.sqrt(d), out=out, work=work)
        assert torch.equal(out, a)


def test_attention_leaves_every_counter_at_zero(ops):
    work, zeroed = ops.paged_attention_workspace(1024, 64, 32, 1, 128), ctypes.c_longlong(0)
    ops.lib().mivgpu_paged_attention_work(1024, 32, 1, ctypes.byref(zeroed))
    assert zeroed.value > 1024
    for name in ATTNS:
        old, new, hq, hkv, d = ATTNS[name]
        q, cache, table, cu, kv = attention_case(ops, old, new, hq, hkv, d)
        ops.paged_attention(q.cuda(), cache, dev(table), dev(cu), dev(kv), hq, hkv, d, 0.1, work=work)
        assert (work[:zeroed.value].view(torch.int32) == 0).all(), name


APPEND_MENDS = {
    "larger": lambda x: x.mul_(2.0 ** 9), "smaller": lambda x: x.mul_(2.0 ** -9), "far larger": lambda x: x.mul_(2.0 ** 40),
    "zeros": lambda x: x.zero_(), "some zeros": lambda x: x[::3].zero_(), "huge V": lambda x: x[:, 6 * 128:].fill_(-3.3e38),
    "NaN in K": lambda x: x[2:70:17, 4 * 128 + 5].fill_(math.nan), "inf in V": lambda x: x[1::9, 7 * 128 + 9].fill_(math.inf),
    "NaN in q": lambda x: x[5, 128 + 3].fill_(math.nan),
}


@pytest.mark.parametrize("name", APPEND_MENDS, ids=list(APPEND_MENDS))
def test_append_of_unusual_values_q_too(ops, name):
    """q of every head whose inputs are finite, whatever stands in the others."""
    old, new, seed, (hq, hkv, d), seen = [7, 100, 0], [3, 1, 75], 5, (4, 2, 128), []

    def mend(x):
        APPEND_MENDS[name](x)
        seen.append(x.clone())
    q_out, _ = check_append(ops, old, new, hq, hkv, d, mend=mend, seed=seed)
    pos, g = layout(old, new, seed)[0], torch.Generator()
    g.manual_seed(seed)                               # the norm's weights, as check_append draws them
    torch.randn(len(pos), (hq + 2 * hkv) * d, generator=g), torch.rand((hq + 2 * hkv) * d, generator=g)
    qw = (1 + 0.1 * torch.randn(d, generator=g)).to(torch.bfloat16)
    x = seen[0][:, :hq * d].double().view(-1, hq, d)
    q, size = oracle.norm_rope(x, qw.double(), pos, THETA, EPS)
    fine = x.isfinite().all(-1)
    got = q_out.cpu().double()
    assert torch.all(((got - q).abs() <= q.abs() * 2.0 ** -8 + size * 2.0 ** -18)[fine])      # as in check_append
    assert got[~fine].isnan().any(-1).all() and int(fine.sum()) >= len(pos) * hq - 1


def test_steps_together_layer_by_layer(ops):
    """As test_steps_together, with each layer's queries kept: both layers' attention is the oracle's."""
    class Keep:
        def __getattr__(self, name):
            return getattr(ops, name)

        def paged_attention(self, q, *args, **kw):
            queries.append(q.clone())
            return ops.paged_attention(q, *args, **kw)

    s = server(ops, 200, 3)
    for new in ([70, 0, 30], [1, 100, 1], [1, 1, 1], [0, 1, 66]):
        s["x"].add_(0.125)
        queries = []
        plan = serve_step(Keep(), s, dev(new), 200)
        n = sum(new)
        assert len(queries) == 2
        for q, cache, att in zip(queries, s["cache"], s["att"]):
            c = to_host(cache)
            for t in (c.k, c.v):
                t.view(torch.uint8).copy_(torch.where((t.view(torch.uint8) & 0x7f) == 0x7f, 0, t.view(torch.uint8)))
            o, size = oracle.attention(q.cpu(), c, host(s["pool"].table), host(plan.cu_q), host(plan.kv_lens), 8, 2, 1 / math.sqrt(128))
            o, size = o.reshape(200, -1), size.reshape(200, -1)
            tol = size * (2.0 ** -8 + 2.0 ** -9) + o.abs() * 2.0 ** -8 + 2.0 ** -100
            assert torch.all((att.cpu().double() - o).abs()[:n] <= tol[:n])
