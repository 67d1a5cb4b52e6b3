"""Precision of paged attention where roundings of one sign add up, against exact results.

Errors of an fp32 score s of a few tens: its product with the scale and log2(e) is rounded twice (2^-24 of it each), ex2.approx
adds 2^-22, the sums a few 2^-24 -- for |s| <= 32 below 32 * 1.45 * 2 * 2^-24 + 2^-21 < 2^-17 of a weight.
"""

import numpy as np
import pytest

from conftest import pkg

pytestmark = pytest.mark.gpu

HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def _dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


@pytest.mark.parametrize("act", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("far", [9, 18, 30])
@pytest.mark.parametrize("batch,kv,length", [(1, 2, 2000), (38, 8, 16384), (1, 1, 60000)])
@pytest.mark.parametrize("dim", [32, 128])
def test_many_small_weights_behind_a_dominating_key(act, far, batch, kv, length, dim):
    """One early key with the score `far` and the value 0, all others with the score 0 and the value 1 (a cluster's call,
    even pieces of more pairs than CTAs, one long context): the result is N e^-far / (1 + N e^-far), within half a step of its
    type (and of the type's smallest number), the weights' own error and their 16-bit parts' (2^-16, bf16)."""
    import torch
    ops, t = pkg("ops"), _dt(act)
    ps = 16
    pages = -(-length // ps)
    k, v = torch.zeros(pages, kv, ps, dim, dtype=t, device="cuda"), torch.ones(pages, kv, ps, dim, dtype=t, device="cuda")
    k[0, :, 3, 0] = far
    v[0, :, 3] = 0
    q = torch.zeros(batch, kv, dim, dtype=t, device="cuda")
    q[..., 0] = 1
    tables = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(batch, 1)   # all requests read one context
    lens = torch.full((batch,), length, dtype=torch.int32, device="cuda")
    out, lse = ops.paged_attention(q, k, v, tables, lens, scale=1.0, return_lse=True)
    rest = (length - 1) * np.exp(-float(far))
    want = rest / (1 + rest)
    tiny = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}[act]
    tol = (HALF[act] + 2.0 ** -17 + (2.0 ** -16 if act == "bf16" else 0)) * want + tiny
    got = out.double().cpu().numpy()
    assert np.abs(got - want).max() <= tol, (got.min(), got.max(), want, tol)
    assert np.abs(lse.double().cpu().numpy() - (far + np.log1p(rest))).max() <= 2.0 ** -17 + 2.0 ** -23 * (far + np.log1p(rest))


@pytest.mark.parametrize("length", [100, 5000, 40000])
def test_fp16_values_of_any_size_and_infinite_ones(length):
    """Equal weights over values from the smallest to the largest fp16 number: their mean; an infinite value stays one."""
    import torch
    ops, ps, dim = pkg("ops"), 16, 64
    pages = -(-length // ps)
    rng = np.random.default_rng(length)
    k = torch.zeros(pages, 1, ps, dim, dtype=torch.float16, device="cuda")
    v = torch.from_numpy(rng.uniform(1, 2, (pages, 1, ps, dim)).astype(np.float32) * 2.0 ** np.linspace(-20, 15, dim).round()).half().cuda()
    v = v.clamp(max=65504.0)
    x = v.permute(0, 2, 1, 3).reshape(-1, dim)[:length].double()
    q = torch.zeros(1, 1, dim, dtype=torch.float16, device="cuda")
    t = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    n = torch.tensor([length], dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, k, v, t, n).double()
    want = x.mean(0)
    # all weights are 1: sums of fp32 products, one of at most 16 keys after the other, then of warps and CTAs
    assert bool(((got - want).abs() <= want * (2.0 ** -11 + 2.0 ** -17) + 2.0 ** -25).all())
    v[length // 2 // ps, 0, length // 2 % ps, 5] = float("inf")
    v[0, 0, 1, 6] = float("nan")
    got2 = ops.paged_attention(q, k, v, t, n)
    assert float(got2[0, 0, 5]) == float("inf") and bool(got2[0, 0, 6].isnan())
    keep = [i for i in range(dim) if i not in (5, 6)]
    assert torch.equal(got2[..., keep].double(), got[..., keep])


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("bf16", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"),
                                       ("bf16", "bf16")])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_one_key_gives_its_value(act, cache, dim):
    """One visible key has the weight 1, so the result is its value: exactly in the 16-bit types; fp32 values enter as two tf32
    parts of 11 bits, the upper one cut off, so that 13 of 24 bits are left, and the lower one rounded to the nearest 11 of
    these: at most half of 2^-21 of the value's power of two is lost, 2^-22 of the value (and the result's own rounding)."""
    import torch
    ops = pkg("ops")
    rng = np.random.default_rng(dim)
    B, H, kv, ps = 40, 6, 2, 16
    x = (rng.normal(size=(B, kv, ps, dim)) * 2.0 ** rng.integers(-12, 12, (B, kv, ps, dim))).astype(np.float32)
    v = torch.from_numpy(x).cuda().to(_dt(cache))
    k = torch.from_numpy(rng.normal(size=(B, kv, ps, dim)).astype(np.float32)).cuda().to(_dt(cache))
    q = torch.from_numpy(rng.normal(size=(B, H, dim)).astype(np.float32)).cuda().to(_dt(act))
    tables = torch.arange(B, dtype=torch.int32, device="cuda")[:, None].contiguous()
    for n, window in ((1, 0), (9, 1), (16, 1)):
        lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
        got = ops.paged_attention(q, k, v, tables, lens, window=window).double()
        want = v[:, :, n - 1].double().repeat_interleave(H // kv, 1)
        tol = (2.0 ** -22 if cache == "f32" else 0.0) + (0.0 if act in (cache, "f32") else HALF[act])
        assert bool(((got - want).abs() <= tol * want.abs()).all()), (n, float(((got - want).abs() / want.abs()).max()))


@pytest.mark.parametrize("length", [1, 7, 100])
def test_fp32_values_are_not_cut_to_one_side(length):
    """Errors of a few keys' results have either sign: over 40 x 6 x 64 results of positive values, each off by at most 2^-22 and
    by 2^-23 on average if all pointed one way, the mean error stays below 2^-24 of the value, the step of an fp32 rounding."""
    import torch
    ops = pkg("ops")
    rng = np.random.default_rng(length)
    B, H, ps, dim = 40, 6, 128, 64
    v = torch.from_numpy(rng.uniform(1, 2, (B, H, ps, dim)).astype(np.float32)).cuda()
    k = torch.zeros_like(v)
    q = torch.zeros(B, H, dim, device="cuda")
    tables = torch.arange(B, dtype=torch.int32, device="cuda")[:, None].contiguous()
    lens = torch.full((B,), length, dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, k, v, tables, lens).double()
    want = v[:, :, :length].double().mean(2)
    assert abs(float(((got - want) / want).mean())) <= 2.0 ** -24
