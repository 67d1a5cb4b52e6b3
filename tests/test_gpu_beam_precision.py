"""The choice's log-sum-exp to 2e-8, whatever the logits look like.

A hypothesis whose score is the negative log-probability of its best token, rounded to fp32, continues to a score next to 0,
which fp32 holds to 2^-24 of itself: it shows the log-sum-exp's error.  Bound: a term is 2^(j/32) * (1 + q), |q| <= 0.022; the
cubic is off by 2.3e-9, its argument by 5 * 2^-31, q by 3 * 2^-24 and 2^(j/32) in fp32 by 2^-23 of 0.022, chains of eight
such products by 5 * 2^-24 of 0.022: below 2e-8 of a sum in which every error has one sign.
"""

import numpy as np
import pytest

from conftest import pkg

import oracle.paged as ref

pytestmark = pytest.mark.gpu

BOUND = 2e-8


def _rows(rng, kind, n, V):
    """Rows of logits: flat tails below one favourite, two levels, normal ones, ones far from 0."""
    x = np.empty((n, V))
    for i in range(n):
        if kind == "tail":
            top, below = rng.uniform(-3, 20), rng.uniform(6, 14)
            x[i] = top - below
            x[i, rng.integers(V)] = top
        elif kind == "levels":
            top = rng.uniform(-3, 20)
            x[i] = top - rng.uniform(8, 20)
            x[i, ::16] = top - rng.uniform(2.1, 8)
            x[i, 7] = top
        elif kind == "normal":
            x[i] = rng.normal(size=V) * rng.uniform(0.1, 6) + rng.uniform(-30, 30)
        elif kind == "far":
            x[i] = rng.uniform(-60000, 60000) + rng.normal(size=V) * 4
        else:
            x[i] = rng.uniform(0.5, 3) * rng.choice([-1e5, 1e5, 1e9]) * (1 + rng.normal(size=V) * 1e-4)
    return x


@pytest.mark.parametrize("act,kind", [(a, k) for a in ("f32", "bf16", "f16") for k in ("tail", "levels", "normal", "far", "huge")
                                      if (a, k) != ("f16", "huge")])   # (beyond fp16)
@pytest.mark.parametrize("V", [500, 6761, 40009, 151936])
def test_log_sum(act, V, kind):
    import torch
    ops = pkg("ops")
    rng = np.random.default_rng(V)
    n = 48
    x = torch.from_numpy(_rows(rng, kind, n, V).astype(np.float32)).cuda()
    x = x.to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[act])
    y = x.double()
    lp = y.amax(-1) - torch.logsumexp(y, -1)
    scores = (-lp).float()
    zero = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    got = ops.beam_select(x[:, None], scores[:, None].contiguous(), zero, zero)
    want = scores.double() + lp
    assert torch.equal(got.tokens[:, 0], (y == y.amax(-1, keepdim=True)).long().argmax(-1))
    err = (got.scores[:, 0].double() - want).abs()
    # (and the 64-bit numbers' own steps where the logits are large: a difference of theirs, its logarithm)
    assert float((err - 2.0 ** -23 * want.abs() - 2.0 ** -50 * y.abs().amax(-1)).max()) <= BOUND, float(err.max())


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("V", [6761, 151936])
def test_close_keys_of_unlike_rows(act, V):
    """A row with a flat tail against one of few near tokens, their best keys 5e-8 to 2e-7 apart: the better one is first."""
    import torch
    rng = np.random.default_rng(3)
    G = 60
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[act]
    grid = lambda a: torch.from_numpy(np.asarray(a, np.float32)).to(dt).double().numpy()  # noqa: E731
    x, s = np.full((G, 2, V), -np.inf), np.zeros((G, 2), np.float32)
    for g in range(G):
        top = float(grid([rng.uniform(2, 20)])[0])
        x[g, 0] = grid([top - np.log(V / rng.uniform(0.3, 2))])[0]
        x[g, 0, rng.integers(V)] = top
        rest = np.exp(x[g, 0].min() - top) * (V - 1)
        m = int(rng.integers(3, 9))                      # near tokens with about the same sum
        x[g, 1, :m] = grid([top + np.log(rest / m)])[0]
        x[g, 1, V - 1] = top
        lp = [-np.log(np.exp(x[g, k] - top).sum()) for k in range(2)]
        s[g, 1] = np.float32(lp[0] - lp[1] + rng.choice([-1, 1]) * rng.uniform(5e-8, 2e-7))
    zero = np.zeros((G, 2), np.int32)
    want = ref.beam(x, s, zero, zero)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    got = pkg("ops").beam_select(cu(x.astype(np.float32)).to(dt), cu(s), cu(zero), cu(zero))
    assert np.array_equal(got.parents.cpu().numpy(), want[1]) and np.array_equal(got.tokens.cpu().numpy(), want[0])
    assert 10 < int((want[1][:, 0] == 0).sum()) < 50


def test_certain_tokens_keep_their_score():
    """A row that allows one token has the log-probability 0, V equal ones -log V: no error at all, so that equal keys of
    unlike rows stay equal (and go to the lower hypothesis)."""
    import torch
    G, K, V = 1, 6, 3000
    x = np.full((G, K, V), -np.inf, np.float32)
    for k, at in enumerate((0.3, -17.25, 1e5, 88.0, -1e9, 3e38)):
        x[0, k, 100 + k] = at
    s, zero = np.full((G, K), -3.7, np.float32), np.zeros((G, K), np.int32)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    ops = pkg("ops")
    got = ops.beam_select(cu(x), cu(s), cu(zero), cu(zero))
    assert got.parents.tolist() == [[0, 1, 2, 3, 4, 5]] and got.tokens.tolist() == [[100 + k for k in range(K)]]
    assert torch.equal(got.scores, cu(s))
    y = np.broadcast_to(np.array([0.3, -17.25, 1e5, 88.0, -1e9, 3e38], np.float32)[None, :, None], (1, K, V))
    got = ops.beam_select(cu(y), cu(s), cu(zero), cu(zero))
    assert got.parents.tolist() == [[0] * K] and got.tokens.tolist() == [list(range(K))]


@pytest.mark.parametrize("score", [-1e30, float(np.finfo(np.float32).min), -1e12])
@pytest.mark.parametrize("K,V", [(2, 300), (4, 6761), (8, 6761), (8, 151936), (20, 40009), (32, 151936)])
def test_scores_that_swallow_the_logits(score, K, V):
    """Hypotheses marked by a huge negative score: all their keys are one number in 64 bits (or nearly), and the tokens are
    still those of the largest logits, the lower hypothesis's first, however the call is cut."""
    import torch
    rng = np.random.default_rng(V + K)
    x = rng.normal(size=(2, K, V)).astype(np.float32)
    x[1] = np.round(x[1] * 2) / 2                     # (equal logits: the lowest tokens)
    s = np.full((2, K), -np.inf, np.float32)
    s[:, K // 2:] = score
    x[0, 0, 5:], s[0, 0] = -np.inf, -1.0              # one hypothesis with five tokens
    zero = np.zeros((2, K), np.int32)
    want = ref.beam(x, s, zero, zero)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    got = pkg("ops").beam_select(cu(x), cu(s), cu(zero), cu(zero))
    assert np.array_equal(got.parents.cpu().numpy(), want[1]) and np.array_equal(got.tokens.cpu().numpy(), want[0])
    if score > -1e20:       # (64 bits next to 1e12 still tell logits 1.2e-4 apart, so other hypotheses may come first)
        return
    assert want[1][1].tolist() == [K // 2] * K
    order = np.lexsort((np.arange(V), -x[1, K // 2].astype(np.float64)))
    assert want[0][1].tolist() == order[:K].tolist()
