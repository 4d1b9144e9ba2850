"""ops.sample against the plain 64-bit definition (tests/paged_oracle.py)."""

import math

import numpy as np
import paged_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from k8s_vgpu_scheduler_amd import ops as o
    from k8s_vgpu_scheduler_amd.utils import build

    build.build_ops()
    o.require_native()
    return o


def check(ops, logits, u, t=None, k=None, p=None, mp=None, work=True):
    """Every row's token is one that the definition gives for a random number within 2^-40 of the one asked."""
    B, V = logits.shape
    f = lambda a, dt: None if a is None else torch.tensor(a, dtype=dt, device="cuda")  # noqa: E731
    args = [f(u, torch.float32), f(t, torch.float32), f(k, torch.int32), f(p, torch.float32), f(mp, torch.float32)]
    tokens, probs = ops.sample(logits, *args, work=ops.sample_workspace(B, V) if work else None)
    rows = logits.double().cpu().numpy()
    get = lambda i, b, d: d if args[i] is None else float(args[i][b].double())  # noqa: E731
    for b in range(B):
        tok, prob = int(tokens[b]), float(probs[b])
        row = rows[b]
        if np.isnan(row).any():
            assert tok == int(np.flatnonzero(np.isnan(row))[0]) and math.isnan(prob)
            continue
        idx, w = oracle.order(row, get(1, b, 1.0), int(get(2, b, 0)), get(3, b, 1.0), get(4, b, 0.0))
        if len(idx) == 0:
            assert tok == -1 and prob == 0.0
            continue
        at = np.flatnonzero(idx == tok)
        assert len(at) == 1, (b, tok, "not kept")
        c, z, x = np.cumsum(w), w.sum(), float(args[0][b].double()) * w.sum()
        at = int(at[0])
        assert w[at] > 0
        # 64-bit sums of up to 2^18 weights, geometric within a value's neighbours: far inside 2^-40
        slack = z * 2.0 ** -40
        last = int(np.flatnonzero(w > 0)[-1])
        assert (c[at] - w[at] <= x + slack) and (x < c[at] + slack or at == last), (b, tok, at)
        assert abs(prob - w[at] / z) <= w[at] / z * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -149
    return tokens, probs


def logits_of(B, V, seed, spread=2.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(B, V, generator=g, device="cuda") * spread
    x[torch.arange(B), torch.randint(0, V, (B,), generator=g, device="cuda")] += 6
    return x.to(torch.bfloat16)


def us(B, seed):
    return np.random.RandomState(seed).rand(B)


@pytest.mark.parametrize("V", [1, 2, 7, 8, 63, 1000, 4096, 32768, 32769, 50257, 151936, 200003])
def test_plain(ops, V):
    check(ops, logits_of(3, V, V), us(3, V))


SETTINGS = {
    "temperature": dict(t=[0.3, 0.7, 1.0, 1.5, 5.0]),
    "top-k": dict(k=[1, 2, 50, 10000, 0]),
    "top-p": dict(p=[0.01, 0.5, 0.9, 0.999, 1.0]),
    "min-p": dict(mp=[0.0, 0.01, 0.1, 0.5, 1.0]),
    "all": dict(t=[0.7, 0.9, 1.2, 0.5, 0.0], k=[50, 20, 1000, 0, 7], p=[0.9, 0.95, 0.8, 0.99, 0.5], mp=[0.05, 0.0, 0.1, 0.02, 0.3]),
    "greedy": dict(t=[0.0, -1.0, 0.0, 0.0, math.nan]),
    "off by value": dict(t=[1.0] * 5, k=[0, -3, 0, 2**31 - 1, -(2**31)], p=[1.0, 2.0, 1.5, math.inf, math.nan], mp=[0.0, -1.0, 0.0, 0.0, 0.0]),
    "extreme": dict(t=[1e-30, 1e30, math.inf, 1e-3, 1.0], p=[0.5, 0.5, 0.5, 0.0, -1.0]),
}


@pytest.mark.parametrize("V", [97, 5000, 151936])
@pytest.mark.parametrize("name", SETTINGS, ids=list(SETTINGS))
def test_settings(ops, name, V):
    for seed in range(3):
        check(ops, logits_of(5, V, seed), us(5, seed + 10), **SETTINGS[name])


@pytest.mark.parametrize("u", [0.0, 0.5, 1.0 - 2.0 ** -24, 1.0, 7.0, math.nan])
def test_random_number_ends(ops, u):
    for V in (5, 4096):
        x = logits_of(2, V, 1)
        tokens, _ = ops.sample(x, torch.full((2,), u, device="cuda"), top_k=torch.tensor([3, 0], dtype=torch.int32, device="cuda"))
        for b, k in enumerate((3, 0)):
            idx, w = oracle.order(x[b].double().cpu().numpy(), 1.0, k, 1.0, 0.0)
            assert int(tokens[b]) in idx
            if u == 0.0:
                assert int(tokens[b]) == idx[0]
            if not u < 1.0:
                assert int(tokens[b]) == idx[-1]


def test_ties_go_to_the_lowest_index(ops):
    x = torch.zeros(4, 3000, dtype=torch.bfloat16, device="cuda")
    x[:, 1::2] = -0.0                                  # equal to +0
    x[1, 700:900] = 1.0
    x[2, 2999] = 1.0
    tokens, _ = check(ops, x, [0.0, 0.0, 0.0, 0.5], t=[0.0, 0.0, 0.0, 1.0])
    assert tokens.tolist() == [0, 700, 2999, 1500]
    tokens, probs = check(ops, x, [0.999] * 4, k=[10, 10, 10, 0], p=[1.0, 1.0, 1.0, 0.5])
    assert tokens.tolist()[:2] == [9, 709] and tokens[3] == 1498


@pytest.mark.parametrize("V", [65535, 65536, 65537, 140000, 151936])
def test_more_equal_values_than_a_counter_holds(ops, V):
    x = torch.full((3, V), 2.5, dtype=torch.bfloat16, device="cuda")
    x[1, ::2] = -1.0
    x[2, V // 2:] = 2.484375                           # its neighbour in the same word
    check(ops, x, [0.0, 0.5, 0.99])
    check(ops, x, [0.9999, 0.75, 0.3], k=[70000, 0, 100000], p=[0.97, 0.5, 0.999])


def test_masked_rows(ops):
    x = logits_of(6, 2000, 5)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 777] = -3.0
    x[2, ::2] = -math.inf
    x[3] = torch.finfo(torch.bfloat16).min
    x[4] = torch.finfo(torch.bfloat16).min
    x[4, 5] = 0.0
    x[5, 3:1999] = -math.inf
    for t in (1.0, 0.0, math.inf):
        tokens, probs = check(ops, x, [0.3] * 6, t=[t] * 6)
        assert tokens[0] == -1 and tokens[1] == 777 and probs[1] == 1.0
        if t == 1.0:
            assert int(tokens[2]) % 2 == 1 and tokens[3] == 600 and tokens[4] == 5


def test_not_finite(ops):
    x = logits_of(4, 1000, 6)
    x[0, 321], x[0, 700] = math.nan, math.nan
    x[1, 20], x[1, 30] = math.inf, math.inf
    x[2, 900] = math.inf
    x[3, 100] = -math.nan
    for t in (1.0, 0.0, math.inf):
        tokens, probs = check(ops, x, [0.7] * 4, t=[t] * 4)
        assert tokens[0] == 321 and tokens[2] == 900 and tokens[3] == 100
        assert tokens[1] == (20 if t == 0.0 else 30)


@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e-3, 1e30])
def test_tiny_and_huge_logits(ops, scale):
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = (torch.randn(4, 3000, generator=g, device="cuda") * scale).to(torch.bfloat16)
    check(ops, x, us(4, 2), t=[scale, 1.0, scale * 0.1, scale], k=[0, 0, 50, 0], p=[1.0, 0.7, 1.0, 0.5])


def test_every_bit_pattern(ops):
    """A row of all bf16 values (without NaN), shuffled."""
    bits = torch.arange(65536, dtype=torch.int32)
    bits = bits[((bits & 0x7f80) != 0x7f80)]
    g = torch.Generator()
    g.manual_seed(0)
    x = bits[torch.randperm(len(bits), generator=g)].to(torch.int16).view(torch.bfloat16)[None].repeat(3, 1).cuda()
    check(ops, x, [0.1, 0.6, 0.9], t=[1e37, 1e38, 1e30], k=[0, 1000, 0])


@pytest.mark.parametrize("lead", range(0, 8))
def test_rows_anywhere_in_memory(ops, lead):
    """Strided rows that start at any bf16: the row's neighbours are never looked at."""
    base = torch.full((5, 1013), 99.0, dtype=torch.bfloat16, device="cuda")
    x = base[:, lead:lead + 1001]
    x.copy_(logits_of(5, 1001, lead))
    tokens, _ = check(ops, x, us(5, lead), t=[0.0, 1.0, 1.0, 0.5, 0.0])
    again, _ = check(ops, x.clone(), us(5, lead), t=[0.0, 1.0, 1.0, 0.5, 0.0])
    assert torch.equal(tokens, again)


@pytest.mark.parametrize("B", [1, 2, 31, 64, 300])
def test_rows(ops, B):
    r = np.random.RandomState(B)
    x = logits_of(B, 20011, B)
    kw = dict(t=r.choice([0.0, 0.7, 1.0], B), k=r.choice([0, 40], B), p=r.choice([1.0, 0.9], B), mp=r.choice([0.0, 0.05], B))
    a, pa = check(ops, x, us(B, B), **kw)
    # a row's answer does not depend on the others beside it
    f = lambda v, dt: torch.tensor(v, dtype=dt, device="cuda")  # noqa: E731
    for b in {0, B // 2, B - 1}:
        t1, p1 = ops.sample(x[b:b + 1], f(us(B, B)[b:b + 1], torch.float32), f(kw["t"][b:b + 1], torch.float32),
                            f(kw["k"][b:b + 1], torch.int32), f(kw["p"][b:b + 1], torch.float32), f(kw["mp"][b:b + 1], torch.float32))
        assert int(t1) == int(a[b]) and float(p1) == float(pa[b])


def test_frequencies(ops):
    """Evenly spread numbers draw each token as often as its probability says, to one in 4096."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]], device="cuda").to(torch.bfloat16).expand(4096, 5).contiguous()
    u = (torch.arange(4096, device="cuda") + 0.5) / 4096
    tokens, _ = ops.sample(x, u)
    want = torch.softmax(x[0].double(), 0) * 4096
    got = torch.bincount(tokens, minlength=5).double()
    assert torch.all((got - want).abs() <= 1.0)


def test_workspace_of_another_kind_is_refused(ops):
    x = logits_of(1, 100, 0)
    for work in (torch.zeros(0, device="cuda"), torch.zeros(0, dtype=torch.int64)):
        with pytest.raises(ValueError, match="sample"):
            ops.sample(x, torch.zeros(1, device="cuda"), work=work)


def test_greedy_is_decode_tail(ops):
    x = logits_of(8, 4096, 9)
    x[3, 1000] = math.nan
    tok = torch.zeros(8, dtype=torch.int64, device="cuda")
    pos, lens = (torch.zeros(8, dtype=torch.int32, device="cuda") for _ in range(2))
    ops.decode_tail(x, tok, pos, lens, ops.decode_tail_workspace(8, "cuda"))
    got, _ = ops.sample(x, torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda"))
    assert torch.equal(tok, got)


def test_captured(ops):
    x = logits_of(4, 151936, 1)
    u, t = torch.rand(4, device="cuda"), torch.full((4,), 0.9, device="cuda")
    tokens, probs = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, device="cuda")
    work = ops.sample_workspace(4, 151936)
    ops.sample(x, u, t, tokens=tokens, probs=probs, work=work)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.sample(x, u, t, tokens=tokens, probs=probs, work=work)
    for i in range(6):
        u.copy_(torch.rand(4, device="cuda"))
        x.copy_(logits_of(4, 151936, i + 2))
        g.replay()
        if i % 2:
            torch.cuda.synchronize()
        want, wp = ops.sample(x, u, t)
        assert torch.equal(tokens, want) and torch.equal(probs, wp)


@pytest.mark.parametrize("mp", [1.0, 1.0000001, 1.5, math.inf])
def test_min_p_above_one_keeps_the_first(ops, mp):
    """No weight reaches a min_p above 1, not the maximum's either: of tied maxima the first is left."""
    x = logits_of(3, 5000, 3)
    x[0, [40, 700, 4999]] = 99.0
    x[1] = 0.5
    for t in (0.5, math.inf):
        tokens, probs = check(ops, x, [0.9] * 3, t=[t] * 3, mp=[mp] * 3)
        if mp > 1:
            assert tokens.tolist() == [40, 0, int(x[2].argmax())] and probs.tolist() == [1.0] * 3
    check(ops, x, [0.9] * 3, k=[2, 10, 2], p=[0.5, 0.9, 1.0], mp=[mp] * 3)
