"""Refusals and host-side parts of the paged 8-bit serving operators (no GPU: every check comes before a launch)."""

import math
from fractions import Fraction

import numpy as np
import paged_oracle as oracle
import pytest
import torch

from k8s_vgpu_scheduler_amd import ops


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def cache(pages=4, hkv=2, d=128):
    return ops.paged_kv_cache(pages, hkv, d, device="cpu")


def test_cache_shapes():
    c = cache(3, 2, 64)
    assert c.k.shape == (3, 2, 64, 64) and c.v.shape == (3, 2, 64, 64) and c.k.dtype == torch.float8_e4m3fn
    c = cache(3, 2, 128)
    assert c.k.shape == (3, 2, 64, 128) and c.v.shape == (3, 2, 128, 64) and c.v_scale.shape == (3, 2)


@pytest.mark.parametrize("args", [(0, 2, 128), (4, 0, 128), (4, 2, 96)])
def test_cache_refuses(args):
    with pytest.raises(ValueError):
        ops.paged_kv_cache(*args, device="cpu")


@pytest.mark.parametrize("args", [(0, 4, 4), (4, 0, 4), (4, 1025, 4), (4, 4, 0)])
def test_pool_refuses(args):
    with pytest.raises(ValueError):
        ops.PagePool(*args, device="cpu")


@pytest.mark.parametrize("d,theta", [(64, 1e4), (128, 1e6)])
def test_rope_turns(d, theta):
    t = ops.rope_turns(theta, d, device="cpu")
    got = t.numpy().view(np.uint64).astype(np.longdouble) / np.longdouble(2) ** 64
    want = np.longdouble(theta) ** (-2 * np.arange(d // 2, dtype=np.longdouble) / d) / (2 * np.longdouble(np.pi))
    # float64 power (the exponent's rounding counts ln(theta) < 14 times) and division: under 2^-48 relative; the
    # table's own rounding to whole 2^-64: half of one
    assert np.all(np.abs(got - want) <= want * 2.0 ** -48 + 2.0 ** -65)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("theta", [1, 1.0, 2.0, 1e4, 5e5, 1e6, 1234567.891, 1e300])
def test_rope_turns_to_half_a_unit(d, theta):
    """An entry t stands for the angle x = theta^(-2i/D) = 2 pi t / 2^64.  x^(D/2) = theta^-i is rational, so that
    t - 1/2 <= 2^64 x / 2 pi <= t + 1/2 is decided in whole numbers, between two fractions of which one is below pi."""
    scale = 10**40
    below = Fraction(31415926535897932384626433832795028841971, scale)
    for i, t in enumerate(ops.rope_turns(theta, d, device="cpu").numpy().view(np.uint64).tolist()):
        want = Fraction(theta) ** -i
        lo, hi = max(Fraction(2 * t - 1, 2), 0), Fraction(2 * t + 1, 2)
        assert (lo * 2 * below / 2**64) ** (d // 2) <= want <= (hi * 2 * (below + Fraction(1, scale)) / 2**64) ** (d // 2), i


@pytest.mark.parametrize("theta,d", [(0.0, 128), (-1.0, 128), (1e6, 96), (math.nan, 128), (math.inf, 128), (1e-300, 128)])
def test_rope_turns_refuses(theta, d):
    with pytest.raises(ValueError):
        ops.rope_turns(theta, d, device="cpu")


PLAN = dict(new_lens=i32(3), lengths=i32(3), table=i32(3, 5), free=i32(7), ring=i32(2), n_tokens=4)


@pytest.mark.parametrize("bad", [
    {},                                                    # on the CPU
    dict(new_lens=i32(4)), dict(new_lens=i32(3).long()), dict(lengths=i32(2)), dict(lengths=i32(6)[::2]),
    dict(table=i32(3)), dict(table=i32(0, 5)), dict(table=i32(3, 0)), dict(table=i32(5, 3).T), dict(free=i32(0)),
    dict(free=i32(1, 7)), dict(ring=i32(3)), dict(n_tokens=-1),
    dict(table=i32(1025, 1), new_lens=i32(1025), lengths=i32(1025)),
    dict(out=ops.PagePlan(i32(3), i32(3), i32(3), i32(4), i32(4))),
    dict(out=ops.PagePlan(i32(4), i32(3), i32(3), i32(4), i32(5))),
])
def test_plan_refuses(bad):
    with pytest.raises(ValueError, match="page_plan"):
        ops.page_plan(**{**PLAN, **bad})


def commit_args(**bad):
    a = dict(plan=ops.PagePlan(i32(4), i32(3), i32(3), i32(4), i32(4)), lengths=i32(3), table=i32(3, 5), free=i32(7),
             ring=i32(2))
    return {**a, **bad}


@pytest.mark.parametrize("bad", [{}, dict(lengths=i32(2)), dict(finished=torch.zeros(3)), dict(ring=i32(1)),
                                 dict(finished=torch.zeros(2, dtype=torch.bool)), dict(table=i32(4, 5)),
                                 dict(plan=ops.PagePlan(i32(4), i32(2), i32(3), i32(4), i32(4)))])
def test_commit_refuses(bad):
    with pytest.raises(ValueError, match="page_commit"):
        ops.page_commit(**commit_args(**bad))


def append_args(**bad):
    a = dict(qkv=bf(3, 8 * 128), q_norm_w=bf(128), k_norm_w=bf(128), positions=i32(3), slots=i32(3),
             turns=torch.zeros(64, dtype=torch.int64), cache=cache(), q_out=bf(3, 4, 128), n_q_heads=4, n_kv_heads=2,
             head_dim=128, eps=1e-6)
    return {**a, **bad}


@pytest.mark.parametrize("bad", [
    {}, dict(qkv=bf(3, 8 * 128).float()), dict(qkv=bf(2, 8 * 128)), dict(qkv=bf(3, 7 * 128)),
    dict(qkv=bf(8 * 128, 3).T), dict(qkv=bf(3, 8 * 128 + 4)[:, :1024]), dict(qkv=bf(1, 1024).expand(3, 1024)),
    dict(q_norm_w=bf(64)), dict(positions=i32(2)), dict(positions=i32(3, 1)), dict(slots=i32(4)),
    dict(slots=i32(3).long()), dict(turns=torch.zeros(32, dtype=torch.int64)), dict(cache=cache(4, 1)),
    dict(cache=cache(4, 2, 64)), dict(q_out=bf(3, 5, 128)), dict(n_q_heads=3), dict(n_kv_heads=0),
    dict(head_dim=96), dict(cache=cache()._replace(v=cache().k)), dict(cache=cache()._replace(k_scale=torch.zeros(4))),
])
def test_append_refuses(bad):
    with pytest.raises(ValueError, match="paged_qk_norm_rope_kv"):
        ops.paged_qk_norm_rope_kv(**append_args(**bad))


def attn_args(**bad):
    a = dict(q=bf(3, 4, 128), cache=cache(), table=i32(2, 3), cu_q=i32(3), kv_lens=i32(2), n_q_heads=4, n_kv_heads=2,
             head_dim=128, scale=0.1, out=bf(3, 512))
    return {**a, **bad}


@pytest.mark.parametrize("bad", [
    {}, dict(q=bf(3, 4, 128).float()), dict(q=bf(3, 5, 128)), dict(q=bf(4, 3, 128).transpose(0, 1)),
    dict(table=i32(2)), dict(table=i32(0, 3)), dict(table=i32(2, 0)), dict(table=i32(1025, 1)), dict(cu_q=i32(2)),
    dict(cu_q=i32(3).long()), dict(kv_lens=i32(3)), dict(out=bf(3, 511)), dict(out=bf(2, 512)), dict(n_q_heads=5),
    dict(head_dim=64), dict(max_new=-1), dict(cache=cache(4, 4)), dict(q=bf(3, 512)), dict(scale=0.0), dict(scale=-0.1),
    dict(scale=math.nan), dict(scale=math.inf), dict(max_new=2**31),
    dict(q=bf(1, 257, 64), cache=cache(1, 257, 64), n_q_heads=257, n_kv_heads=257, head_dim=64, out=bf(1, 257 * 64)),
])
def test_attention_refuses(bad):
    with pytest.raises(ValueError, match="paged_attention"):
        ops.paged_attention(**attn_args(**bad))


@pytest.mark.parametrize("scale", [0.0, -1.0, 1e-50, 2.0 ** -127, 2.0 ** 127, 1e39, math.inf, math.nan])
def test_attention_refuses_scales_that_fp32_lacks(scale):
    """As fp32 these are 0 or infinite: 0 times a masked score's -inf would be NaN."""
    with pytest.raises(ValueError, match="paged_attention: q must be .* scale"):
        ops.paged_attention(**attn_args(scale=scale))


@pytest.mark.parametrize("scale", [2.0 ** -126, 1e-30, 1, 1e30, 2.0 ** 126])
def test_attention_takes_scales_that_fp32_has(scale):
    with pytest.raises(ValueError, match="on one GPU"):
        ops.paged_attention(**attn_args(scale=scale))


@pytest.mark.parametrize("args", [(-1, 1, 4, 2, 128), (2**31, 1, 4, 2, 128), (1, 0, 4, 2, 128), (1, 1025, 4, 2, 128), (1, 1, 5, 2, 128),
                                  (1, 1, 4, 0, 128), (1, 1, 257, 257, 64), (1, 1, 4, 2, 96)])
def test_attention_workspace_refuses(args):
    with pytest.raises(ValueError, match="paged_attention_workspace"):
        ops.paged_attention_workspace(*args, device="cpu")


def sample_args(**bad):
    a = dict(logits=bf(2, 10), uniform=torch.zeros(2), temperature=torch.zeros(2), top_k=i32(2), top_p=torch.zeros(2),
             min_p=torch.zeros(2))
    return {**a, **bad}


@pytest.mark.parametrize("bad", [
    {}, dict(logits=bf(10)), dict(logits=bf(2, 10).float()), dict(logits=bf(10, 2).T), dict(logits=bf(0, 10)),
    dict(logits=bf(2, 0)), dict(logits=bf(1, 10).expand(2, 10)), dict(uniform=torch.zeros(3)),
    dict(uniform=torch.zeros(2).double()), dict(temperature=torch.zeros(1)), dict(top_k=torch.zeros(2)),
    dict(top_p=torch.zeros(2, 1)), dict(min_p=torch.zeros(4)[::2]), dict(tokens=i32(2)), dict(probs=torch.zeros(3)),
])
def test_sample_refuses(bad):
    with pytest.raises(ValueError, match="sample"):
        ops.sample(**sample_args(**bad))


@pytest.mark.parametrize("args", [(0, 10), (1, 0), (1, 128 * 32768 + 1)])
def test_sample_workspace_refuses(args):
    with pytest.raises(ValueError, match="sample_workspace"):
        ops.sample_workspace(*args, device="cpu")


def test_oracle_plan_by_hand():
    """Two requests, one page short: the second is refused, the third needs none."""
    table = np.full((3, 4), -1)
    table[0, 0], table[2, 0] = 9, 8
    got = oracle.plan([70, 65, 1], [10, 0, 3], table, np.arange(10), [9, 2], 136)
    assert got["taken"].tolist() == [1, -1, 0] and got["kv_lens"].tolist() == [80, 0, 4]
    assert got["table"][0].tolist() == [9, 9, -1, -1] and got["slots"][0] == 9 * 64 + 10
    assert got["slots"][54] == 9 * 64 and got["slots"][70] == -1 and got["slots"][135] == 8 * 64 + 3
    assert got["positions"][135] == 3 and got["cu_q"].tolist() == [0, 70, 135, 136]


def test_oracle_sample_by_hand():
    row = np.log(np.array([0.1, 0.4, 0.1, 0.4]))
    idx, w = oracle.order(row, 1.0, 0, 1.0, 0.0)
    assert idx.tolist() == [1, 3, 0, 2] and np.allclose(w, [1, 1, 0.25, 0.25])
    assert oracle.order(row, 1.0, 3, 1.0, 0.0)[0].tolist() == [1, 3, 0]
    assert oracle.order(row, 1.0, 0, 0.79, 0.0)[0].tolist() == [1, 3]
    assert oracle.order(row, 1.0, 0, 0.81, 0.0)[0].tolist() == [1, 3, 0]
    assert oracle.order(row, 1.0, 0, 1.0, 0.3)[0].tolist() == [1, 3]
    assert oracle.order(row, 0.0, 0, 1.0, 0.0)[0].tolist() == [1]


def test_oracle_scale():
    for amax, e in ((448.0, 0), (448.001, 1), (224.0, -1), (1.0, -8), (0.0, oracle.EMIN), (3e38, oracle.EMAX)):
        assert oracle.scale_for(amax) == 2.0 ** e
