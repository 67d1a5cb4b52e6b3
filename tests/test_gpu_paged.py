"""The paged-cache and beam-search operators against the oracle's 64-bit restatement.

Tolerances.  fp32 attention: a score is a dot product of up to 128 terms whose partial sums stay
below ~4, so its rounding error is about sqrt(128) * 4 * 2^-24 = 3e-6, which is the relative error of
a weight; exp and the sums add a few 2^-24, and errors of different keys average out: 1e-5 of a
row's largest value, as the suite holds its other fp32 operators to.  16-bit outputs add half a step
of the value (2^-8 bf16, 2^-11 fp16).  RoPE: two products and a sum, 3 * 2^-24 of the terms' size.
Pages, slots, tokens and copies are exact.
"""

import numpy as np
import pytest

from conftest import pkg

import oracle.paged as ref

pytestmark = pytest.mark.gpu

STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _ops():
    return pkg("ops")


def _dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _cuda(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _np(t):
    return t.float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _tables(rng, lens, ps, cols, extra=3):
    """Distinct random pages for every request; -1 behind them.  Returns (tables, pages in the pool)."""
    held = [-(-n // ps) for n in lens]
    P = sum(held) + extra
    ids = rng.permutation(P).astype(np.int32)
    t, at = np.full((len(lens), cols), -1, np.int32), 0
    for b, h in enumerate(held):
        t[b, :h] = ids[at:at + h]
        at += h
    return t, P, ids[at:]


# ---------------------------------------------------------------------------
# block tables and slots
# ---------------------------------------------------------------------------

def _extend_both(lens, new, tables, stack, count, ps, T, release):
    ops = _ops()
    want = ref.extend(lens, new, tables, stack, count, ps, T, release)
    td, sd = _cuda(tables), _cuda(stack)
    ld, cd = _cuda(lens), _cuda(np.array([count], np.int32))
    got = ops.paged_extend(ld, _cuda(new), td, sd, cd, ps, T, release=None if release is None else _cuda(release))
    used = want[1][:want[7]]
    assert np.array_equal(_np(td), want[0])
    assert int(got.free_count) == want[7] and np.array_equal(_np(sd)[:want[7]], used)
    for a, b in zip((got.slots, got.seq, got.pos, got.offsets, got.lens), want[2:7]):
        assert np.array_equal(_np(a), b)
    assert np.array_equal(_np(ld), lens) and int(cd) == count     # the inputs stay
    return got


@pytest.mark.parametrize("batch", [1, 2, 33, 1024, 1025, 2500])
@pytest.mark.parametrize("ps", [1, 7, 16])
@pytest.mark.parametrize("kind", ["decode", "prefill", "short", "release"])
def test_extend(batch, ps, kind):
    rng = np.random.default_rng(batch * 31 + ps)
    lens = rng.integers(0, 40, batch).astype(np.int32)
    new = rng.integers(0, 2 if kind == "decode" else 30, batch).astype(np.int32)
    cols = -(-70 // ps)
    tables, P, rest = _tables(rng, lens, ps, cols, extra=int(-(-lens.sum() // ps)) + 30 * batch)
    if kind == "short":
        rest = rest[:len(rest) // 9]
    stack = np.full(P, -7, np.int32)
    stack[:len(rest)] = rest
    release = (rng.random(batch) < 0.4).astype(np.int32) * 5 if kind == "release" else None
    T = int(new.sum()) + (5 if kind != "short" else 0)
    _extend_both(lens, new, tables, stack, len(rest), ps, T, release)


def test_extend_edges():
    """No requests, no new tokens, negative numbers, too few rows or columns, an empty stack, a count
    beyond the stack."""
    e = np.zeros(0, np.int32)
    _extend_both(e, e, np.zeros((0, 3), np.int32), np.arange(4, dtype=np.int32), 4, 16, 3, None)
    _extend_both(e, e, np.zeros((0, 0), np.int32), np.zeros(0, np.int32), 0, 16, 0, None)
    z = np.array([0, 5, -3], np.int32)
    t = np.array([[-1, -1], [9, -1], [-1, -1]], np.int32)
    s = np.arange(8, dtype=np.int32)
    _extend_both(z, np.array([0, -2, 3], np.int32), t, s, 6, 4, 9, None)
    _extend_both(z, np.array([2, 3, 3], np.int32), t, s, 6, 4, 4, None)       # rows: the second does not fit
    _extend_both(z, np.array([9, 1, 1], np.int32), t, s, 6, 4, 40, None)      # columns: the first does not fit
    _extend_both(z, np.array([1, 1, 1], np.int32), t, s, 0, 4, 40, None)      # no page left
    _extend_both(z, np.array([1, 1, 1], np.int32), t, s, 0, 4, 40, np.array([0, 1, 0], np.int32))
    _extend_both(z, np.array([1, 1, 1], np.int32), t, s, 99, 4, 40, None)


@pytest.mark.parametrize("batch,T", [(3, 50000), (700, 60000)])
def test_extend_long_prompts(batch, T):
    rng = np.random.default_rng(T)
    lens = rng.integers(0, 50, batch).astype(np.int32)
    new = rng.integers(0, 2 * T // batch, batch).astype(np.int32)
    cols = int(-(-(lens + new).max() // 16))
    tables, P, rest = _tables(rng, lens, 16, cols, extra=T // 16 + 2 * batch)
    stack = np.zeros(P, np.int32)
    stack[:len(rest)] = rest
    _extend_both(lens, new, tables, stack, len(rest), 16, T, None)


def test_extend_in_place_and_wide_table():
    """The state advanced in place through ``out``, and a table that is a slice of a wider one."""
    import torch
    ops = _ops()
    rng = np.random.default_rng(4)
    lens = rng.integers(0, 20, 40).astype(np.int32)
    tables, P, rest = _tables(rng, lens, 4, 12, extra=300)
    stack = np.zeros(P, np.int32)
    stack[:len(rest)] = rest
    wide = torch.full((40, 19), -9, dtype=torch.int32, device="cuda")
    view = wide[:, 3:15]
    view.copy_(_cuda(tables))
    ld, cd, sd = _cuda(lens), _cuda(np.array([len(rest)], np.int32)), _cuda(stack)
    out = ops.PagedStep(*(torch.empty(n, dtype=t, device="cuda") for n, t in
                          ((60, torch.int64), (60, torch.int32), (60, torch.int32), (41, torch.int32))), ld, cd)
    count = len(rest)
    for step in range(9):
        new = rng.integers(0, 3, 40).astype(np.int32)
        rel = (rng.random(40) < 0.2).astype(np.int32)
        tables, stack, slots, seq, pos, offsets, lens, count = ref.extend(lens, new, tables, stack, count, 4, 60, rel)
        ops.paged_extend(ld, _cuda(new), view, sd, cd, 4, 60, release=_cuda(rel), out=out)
        assert np.array_equal(_np(view), tables) and np.array_equal(_np(ld), lens) and int(cd) == count, step
        assert np.array_equal(_np(out.slots), slots) and np.array_equal(_np(out.offsets), offsets)
    assert bool((wide[:, :3] == -9).all()) and bool((wide[:, 15:] == -9).all())


def test_extend_many_requests_in_place():
    """Hundreds of requests that come, grow and go, the state advanced in place; twice the same bits."""
    import torch
    ops = _ops()
    rng = np.random.default_rng(40)
    B, ps, cols, P = 300, 4, 40, 9000
    for repeat in range(2):
        rng = np.random.default_rng(40)
        tables, stack = np.full((B, cols), -1, np.int32), np.arange(P, dtype=np.int32)
        lens, count = np.zeros(B, np.int32), P
        td, sd, ld, cd = _cuda(tables), _cuda(stack), _cuda(lens), _cuda(np.array([count], np.int32))
        out = ops.PagedStep(*(torch.empty(n, dtype=t, device="cuda") for n, t in
                              ((5000, torch.int64), (5000, torch.int32), (5000, torch.int32), (B + 1, torch.int32))), ld, cd)
        for step in range(6):
            new = rng.integers(0, 30, B).astype(np.int32)
            rel = (rng.random(B) < 0.3).astype(np.int32)
            tables, stack, slots, seq, pos, offsets, lens, count = ref.extend(lens, new, tables, stack, count, ps, 5000, rel)
            ops.paged_extend(ld, _cuda(new), td, sd, cd, ps, 5000, release=_cuda(rel), out=out)
            for a, b in ((td, tables), (ld, lens), (out.slots, slots), (out.seq, seq), (out.pos, pos), (out.offsets, offsets)):
                assert np.array_equal(_np(a), b), step
            assert int(cd) == count and np.array_equal(_np(sd)[:count], stack[:count])


# ---------------------------------------------------------------------------
# RoPE and store
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"),
                                       ("bf16", "f32")])
@pytest.mark.parametrize("rows,heads,kv,dim,ps", [(1, 14, 2, 64, 16), (37, 4, 4, 32, 5), (9, 3, 1, 96, 1),
                                                  (1300, 32, 8, 128, 64), (5, 6, 2, 16, 8), (3, 2, 1, 256, 4)])
@pytest.mark.parametrize("layout", ["head", "row"])
def test_append(act, cache, rows, heads, kv, dim, ps, layout):
    import torch
    ops = _ops()
    rng = np.random.default_rng(rows + dim)
    P, npos = -(-rows // ps) + 4, 100
    wide = _cuda(rng.normal(size=(rows, (heads + 2 * kv) * dim + 16)).astype(np.float32), _dt(act))
    qkv = wide[:, :-16] if layout == "row" else wide[:, :-16].contiguous()
    slots = rng.permutation(P * ps)[:rows].astype(np.int64)
    if rows > 2:
        slots[1] = -1
    pos = rng.integers(0, npos, rows).astype(np.int32)
    ang = rng.uniform(0, 6.2, size=(npos, dim // 2))
    ang = np.concatenate([ang, ang], 1)
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    pools = []
    for _ in range(2):
        shape = (P, kv, ps, dim) if layout == "head" else (P, ps, kv, dim)
        t = _cuda(rng.normal(size=shape).astype(np.float32), _dt(cache))
        pools.append(t if layout == "head" else t.transpose(1, 2))
    before = [_np(t) for t in pools]
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = ops.paged_append(qkv, _cuda(slots), _cuda(pos), pools[0], pools[1], heads, _cuda(cos), _cuda(sin), bad=bad)
    x = _np(qkv).reshape(rows, heads + 2 * kv, dim)
    turned = ref.rope_rows(x[:, :heads + kv], cos[pos], sin[pos])
    size = np.abs(x[:, :heads + kv]) + np.abs(np.roll(x[:, :heads + kv], dim // 2, -1))

    def near(got, want, term, step):
        assert np.all(np.abs(got - want) <= 3 * 2.0 ** -24 * term + step * np.abs(want) * (step > 2.0 ** -24) + 1e-7 * (step > 2.0 ** -24))

    near(_np(q), turned[:, :heads], size[:, :heads], STEP[act])
    keep = slots >= 0
    page, row = slots[keep] // ps, slots[keep] % ps
    k, v = _np(pools[0]), _np(pools[1])
    near(k[page, :, row], turned[keep, heads:], size[keep, heads:], STEP[cache])
    assert np.array_equal(v[page, :, row], _np(_cuda(x[keep, heads + kv:]).to(_dt(cache))))
    untouched = np.ones((P, ps), bool)
    untouched[page, row] = False
    for now, was in zip((k, v), before):
        assert np.array_equal(now.transpose(0, 2, 1, 3)[untouched], was.transpose(0, 2, 1, 3)[untouched])
    assert int(bad) == 0


def test_append_without_rotation_and_outside():
    """No tables: q and k as they are; slots outside the pool and positions outside the tables store
    nothing and are counted."""
    import torch
    ops = _ops()
    rng = np.random.default_rng(1)
    qkv = _cuda(rng.normal(size=(6, 8 * 32)).astype(np.float32))
    k, v = torch.zeros(3, 2, 4, 32, device="cuda"), torch.zeros(3, 2, 4, 32, device="cuda")
    slots = _cuda(np.array([3, -1, 12, -2, 1 << 40, 11], np.int64))
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = ops.paged_append(qkv, slots, None, k, v, 4, bad=bad)
    x = qkv.view(6, 8, 32)
    assert torch.equal(q, x[:, :4]) and int(bad) == 3
    assert torch.equal(k[0, :, 3], x[0, 4:6]) and torch.equal(v[2, :, 3], x[5, 6:])
    assert int(torch.count_nonzero(k.abs().sum((1, 3)))) == 2
    cos, sin = torch.ones(5, 32, device="cuda"), torch.zeros(5, 32, device="cuda")
    k.zero_()
    ops.paged_append(qkv, _cuda(np.arange(6, dtype=np.int64)), _cuda(np.array([0, 4, 5, -1, 2, 9], np.int32)), k, v, 4, cos,
                     sin, bad=bad)
    assert int(bad) == 6 and int(torch.count_nonzero(k.abs().sum((1, 3)))) == 3


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _attention(rng, lens, heads, kv, dim, ps, act="f32", cache="f32", window=0, layout="head", cols=None, holes=0):
    import torch
    ops = _ops()
    B = len(lens)
    cols = max(1, max(-(-n // ps) for n in lens)) if cols is None else cols
    tables, P, rest = _tables(rng, lens, ps, cols)
    pools = []
    for _ in range(2):
        a = rng.normal(size=(P, kv, ps, dim)).astype(np.float32)
        for b, n in enumerate(lens):      # what lies behind the last token is not part of the request
            if n % ps:
                a[tables[b, n // ps], :, n % ps:] = np.nan
        a[rest] = np.inf
        t = _cuda(a, _dt(cache))
        pools.append(t if layout == "head" else t.transpose(1, 2).contiguous().transpose(1, 2))
    for i in range(holes):
        b = int(rng.integers(B))
        if lens[b]:
            tables[b, int(rng.integers(-(-lens[b] // ps)))] = [-1, P, 1 << 30, -(1 << 31)][i % 4]
    wide = _cuda(rng.normal(size=(B, heads + 3, dim)).astype(np.float32), _dt(act))
    q = wide[:, 1:1 + heads] if layout == "row" else wide[:, :heads].contiguous()
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = ops.paged_attention(q, pools[0], pools[1], _cuda(tables), _cuda(np.array(lens, np.int32)), window=window,
                                   return_lse=True, bad=bad)
    scale = 1.0 / np.sqrt(dim)
    want, wl = ref.attention(_np(q), _np(pools[0]), _np(pools[1]), tables, lens, scale, window)
    got, gl = _np(out).astype(np.float64), _np(lse)
    big = np.abs(want).max(-1, keepdims=True)
    step = STEP[act] if act != "f32" else 0.0
    assert np.all(np.abs(got - want) <= step * np.abs(want) + 1e-5 * big + (1e-7 if act == "f16" else 0))
    assert np.array_equal(np.isinf(gl), np.isinf(wl))
    fin = np.isfinite(wl)
    assert np.all(np.abs(gl[fin] - wl[fin]) <= 1e-5 * np.maximum(1, np.abs(wl[fin])))
    first = [max(0, n - window) // ps if window else 0 for n in lens]
    holes_seen = sum(int(((tables[b, first[b]:-(-n // ps)] < 0) | (tables[b, first[b]:-(-n // ps)] >= P)).sum())
                     for b, n in enumerate(lens))
    assert int(bad) == holes_seen
    return out


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"),
                                       ("bf16", "f32")])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (8, 8, 32), (3, 1, 96), (32, 4, 128), (16, 1, 64), (40, 2, 128)])
def test_attention_types_and_heads(act, cache, heads, kv, dim):
    rng = np.random.default_rng(heads * dim)
    _attention(rng, [1, 0, 17, 130, 64, 333, 16, 15], heads, kv, dim, 16, act, cache)


@pytest.mark.parametrize("ps", [1, 3, 8, 16, 24, 32, 100])
@pytest.mark.parametrize("layout", ["head", "row"])
def test_attention_page_sizes_and_layouts(ps, layout):
    rng = np.random.default_rng(ps)
    _attention(rng, [0, 1, 2, 15, 16, 17, 127, 128, 129, 700], 14, 2, 64, ps, layout=layout)
    _attention(rng, [5, 300], 6, 3, 128, ps, "bf16", "bf16", layout=layout)


@pytest.mark.parametrize("window", [1, 5, 16, 100, 128, 5000])
@pytest.mark.parametrize("ps", [16, 24, 7])
def test_attention_window(window, ps):
    rng = np.random.default_rng(window)
    _attention(rng, [0, 1, 15, 16, 100, 129, 1000], 14, 2, 64, ps, window=window)
    _attention(rng, [2000], 4, 4, 32, ps, "f32", "f16", window=window)


@pytest.mark.parametrize("batch", [1, 2, 5])
@pytest.mark.parametrize("length", [2048, 5000, 20001])
@pytest.mark.parametrize("cache,dim", [("f32", 64), ("bf16", 128)])
def test_attention_long(batch, length, cache, dim):
    rng = np.random.default_rng(length + batch)
    _attention(rng, [max(length - 777 * b, 0) for b in range(batch)], 4, 2, dim, 16, "f32", cache)


def test_attention_many_requests():
    rng = np.random.default_rng(77)
    _attention(rng, rng.integers(0, 60, 1500).tolist(), 4, 2, 32, 16)
    _attention(rng, [0] * 40 + [900] + [0] * 500 + [3], 14, 2, 64, 16)
    _attention(rng, [0, 0, 0], 14, 2, 64, 16, cols=4)


def test_attention_holes_and_clipped_lengths():
    """Page numbers outside the pool hide their tokens (a request may be left with none), lengths
    beyond the table count as its columns, negative ones as none."""
    import torch
    rng = np.random.default_rng(8)
    _attention(rng, [400, 10, 700, 33], 14, 2, 64, 16, holes=12)
    _attention(rng, [400, 10, 700, 33], 3, 3, 128, 5, "bf16", "bf16", holes=30)
    _attention(rng, [16, 3], 4, 2, 64, 16, holes=8)
    ops = _ops()
    k = _cuda(rng.normal(size=(4, 2, 8, 64)).astype(np.float32))
    q = _cuda(rng.normal(size=(3, 4, 64)).astype(np.float32))
    t = _cuda(np.array([[0, 1], [2, 3], [1, 2]], np.int32))
    got = ops.paged_attention(q, k, k, t, _cuda(np.array([16, 99, -4], np.int32)))
    want = ops.paged_attention(q, k, k, t, _cuda(np.array([16, 16, 0], np.int32)))
    assert torch.equal(got, want) and not bool(got[2].any())


def test_attention_extreme_values():
    """Scores of +-1e4 (softmax of one key), keys of -inf scores (all of them: zeros), infinite and
    NaN values of visible tokens stay what they are in the formula."""
    import torch
    ops = _ops()
    rng = np.random.default_rng(3)
    k = rng.normal(size=(40, 1, 16, 64)).astype(np.float32) * 300
    v = rng.normal(size=(40, 1, 16, 64)).astype(np.float32)
    t = rng.permutation(40).astype(np.int32).reshape(1, 40)
    q = rng.normal(size=(1, 2, 64)).astype(np.float32) * 30
    got = ops.paged_attention(_cuda(q), _cuda(k), _cuda(v), _cuda(t), _cuda(np.array([640], np.int32)), scale=1.0)
    want, _ = ref.attention(q, k, v, t, [640], 1.0)
    assert np.abs(_np(got) - want).max() <= 1e-4 * np.abs(want).max()
    kk = np.full((1, 1, 16, 64), 0, np.float32)
    kk[0, 0, :, 0] = -np.inf
    q1 = np.ones((1, 1, 64), np.float32)
    one = np.zeros((1, 1), np.int32)
    got, lse = ops.paged_attention(_cuda(q1), _cuda(kk), _cuda(v[:1]), _cuda(one), _cuda(np.array([9], np.int32)),
                                   return_lse=True)
    assert not bool(got.any()) and float(lse) == -np.inf
    kk[0, 0, 4, 0] = 0
    vv = v[:1].copy()
    vv[0, 0, 4, 3] = np.inf
    got = ops.paged_attention(_cuda(q1), _cuda(kk), _cuda(vv), _cuda(one), _cuda(np.array([5], np.int32)))
    # one key counts, so the result is its value; values enter the products as two tf32 parts: what the upper part
    # (11 bits) leaves is below 2^-10 of the value and keeps 11 bits itself, so less than 2^-20 of the value is lost
    assert float(got[0, 0, 3]) == np.inf and np.all(np.abs(_np(got)[0, 0, 4:] - vv[0, 0, 4, 4:]) <= 2.0 ** -20 * np.abs(vv[0, 0, 4, 4:]))
    kk[0, 0, 2, 5] = np.nan
    got = ops.paged_attention(_cuda(q1), _cuda(kk), _cuda(vv), _cuda(one), _cuda(np.array([5], np.int32)))
    assert bool(got.isnan().all())


def test_attention_repeats_and_out():
    """The same call twice gives the same bits; ``out`` receives the result."""
    import torch
    ops = _ops()
    rng = np.random.default_rng(5)
    lens = [9000, 20, 1, 4000]
    tables, P, _ = _tables(rng, lens, 16, 600)
    k, v = (_cuda(rng.normal(size=(P, 2, 16, 64)).astype(np.float32)) for _ in range(2))
    q = _cuda(rng.normal(size=(4, 14, 64)).astype(np.float32))
    a = (_cuda(tables), _cuda(np.array(lens, np.int32)))
    one = ops.paged_attention(q, k, v, *a)
    out = torch.empty_like(q)
    for _ in range(3):
        assert ops.paged_attention(q, k, v, *a, out=out) is out and torch.equal(out, one)


def test_attention_far_pages():
    """Element offsets past 2^32 in a pool of more than 8 GB (bf16)."""
    import torch
    ops = _ops()
    P = (1 << 32) // (8 * 16 * 128) + 9
    k = torch.zeros(P, 8, 16, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(P, 8, 16, 128, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(6)
    qkv = _cuda(rng.normal(size=(32, 48 * 128)).astype(np.float32)).bfloat16()
    pages = np.array([[P - 1, P - 7]], np.int32)
    slots = (pages[0][:, None].astype(np.int64) * 16 + np.arange(16)).reshape(-1)
    ops.paged_append(qkv, _cuda(slots), None, k, v, 32)
    q = qkv[:1, :32 * 128].view(1, 32, 128)
    got = ops.paged_attention(q, k, v, _cuda(pages), _cuda(np.array([32], np.int32)))
    small = torch.stack([k[P - 1], k[P - 7]]), torch.stack([v[P - 1], v[P - 7]])
    want = ops.paged_attention(q, *small, _cuda(np.array([[0, 1]], np.int32)), _cuda(np.array([32], np.int32)))
    assert torch.equal(got, want) and bool(small[0].any())


# ---------------------------------------------------------------------------
# beams
# ---------------------------------------------------------------------------

def _beam(logits, scores, counts, done, stop=None, min_len=None, alpha=0.0, act="f32"):
    ops = _ops()
    ld = _cuda(logits, _dt(act))
    got = ops.beam_select(ld, _cuda(scores), _cuda(counts), _cuda(done), stop=stop,
                          min_len=None if min_len is None else _cuda(min_len), length_penalty=alpha)
    want = ref.beam(_np(ld), scores, counts, done, stop or (0, 0), min_len, alpha)
    for name, a, b in zip(("tokens", "parents"), (got.tokens, got.parents), want):
        assert np.array_equal(_np(a), b), (name, _np(a), b)
    assert np.array_equal(_np(got.counts), want[3]) and np.array_equal(_np(got.done), want[4])
    s, w = _np(got.scores), want[2]
    assert np.array_equal(np.isinf(s), np.isinf(w))
    fin = np.isfinite(w)
    assert np.all(np.abs(s[fin] - w[fin]) <= 2.0 ** -23 * np.abs(w[fin]) + 1e-30)
    return got


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_beam_one_hypothesis_of_several(act):
    """A view of every group's third row: its rows are a group's logits apart."""
    import torch
    ops, rng = _ops(), np.random.default_rng(77)
    x = _cuda(rng.normal(size=(3, 5, 1111)).astype(np.float32) * 3, _dt(act))
    z, s = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.zeros(3, 1, device="cuda")
    got, want = ops.beam_select(x[:, 2:3], s, z, z), ops.beam_select(x[:, 2:3].contiguous(), s, z, z)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(x[:, 2].gather(1, got.tokens)[:, 0], x[:, 2].amax(-1))


def _state(rng, G, K, fin=0.2):
    counts = np.repeat(rng.integers(1, 30, (G, 1)), K, 1).astype(np.int32)
    done = (rng.random((G, K)) < fin).astype(np.int32)
    counts -= done * rng.integers(0, 2, (G, K)).astype(np.int32)
    scores = (-2.0 * counts * rng.uniform(0.7, 1.3, (G, K))).astype(np.float32)
    return scores, counts, done


@pytest.mark.parametrize("G,K,V", [(1, 1, 1), (1, 1, 6761), (3, 4, 6761), (1, 2, 1), (2, 5, 3), (4, 32, 40), (2, 16, 4096),
                                   (2, 32, 4097), (9, 8, 20011), (1, 7, 151936), (40, 3, 33)])
@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("alpha", [0.0, 0.7])
def test_beam(G, K, V, act, alpha):
    rng = np.random.default_rng(G * K + V)
    logits = (rng.normal(size=(G, K, V)) * 3).astype(np.float32)
    scores, counts, done = _state(rng, G, K)
    stop = (V - V // 8, V) if V > 8 else None
    _beam(logits, scores, counts, done, stop, rng.integers(0, 30, G).astype(np.int32), alpha, act)


@pytest.mark.parametrize("G,K,V", [(1, 32, 700), (2, 32, 6761), (1, 32, 40009), (2, 20, 30001), (1, 12, 100000), (1, 3, 140000)])
@pytest.mark.parametrize("kind", ["plain", "ties", "one", "rising", "flat", "banned"])
def test_beam_few_tiles_and_many_candidates(G, K, V, kind):
    """Chunks with fewer tiles than hypotheses and rows of many chunks: ties everywhere, all winners in one
    row, in its last tile or chunk, every logit near the maximum, the best tokens not allowed yet."""
    rng = np.random.default_rng(V + K)
    x = (rng.normal(size=(G, K, V)) * 3).astype(np.float32)
    scores, counts, done = _state(rng, G, K)
    stop = min_len = None
    if kind == "ties":
        x = np.round(x / 2) * 2
        scores, counts, done = np.zeros_like(scores), np.ones_like(counts), done * 0
    elif kind == "one":
        scores -= 50
        scores[:, K // 2], done[:, K // 2] = 0, 0
    elif kind == "rising":
        x = np.sort(x, -1)
    elif kind == "flat":
        x = (x / 8 - 4).astype(np.float32)
    elif kind == "banned":
        stop, min_len = (V // 3, V - 5), np.full(G, 100, np.int32)
        x[:, :, V // 3:V - 5] += 9
        x[:, 0, :V // 3] = -np.inf
    _beam(x, scores, counts, done, stop, min_len, 0.6)


def test_beam_first_step_and_ties():
    """Only the first hypothesis exists at the start; equal keys go to the lower hypothesis, then token."""
    rng = np.random.default_rng(2)
    G, K, V = 2, 6, 500
    logits = np.repeat(rng.normal(size=(G, 1, V)), K, 1).astype(np.float32)
    scores = np.full((G, K), -np.inf, np.float32)
    scores[:, 0] = 0
    zero = np.zeros((G, K), np.int32)
    got = _beam(logits, scores, zero, zero)
    assert np.all(_np(got.parents) == 0)
    _beam(logits, np.zeros((G, K), np.float32), zero, zero)                # every beam alike
    _beam(np.zeros((G, K, V), np.float32), np.zeros((G, K), np.float32), zero, zero)
    _beam(np.where(rng.random((G, K, V)) < 0.5, 0.0, -0.0).astype(np.float32), np.zeros((G, K), np.float32), zero, zero)
    up = np.sort(rng.normal(size=(G, K, 9000)), -1).astype(np.float32)     # every token better than the last
    _beam(up, np.zeros((G, K), np.float32), zero, zero)
    _beam(up[..., ::-1].copy(), np.zeros((G, K), np.float32), zero, zero)


def test_beam_masks_infinities_and_nan():
    """Rows of -inf, NaN logits and scores, +inf logits, all tokens stop ids, too few candidates, all
    hypotheses finished."""
    rng = np.random.default_rng(12)
    G, K, V = 3, 4, 300
    zero = np.zeros((G, K), np.int32)
    x = rng.normal(size=(G, K, V)).astype(np.float32)
    s = rng.normal(size=(G, K)).astype(np.float32)
    y = x.copy()
    y[0, 1] = -np.inf
    y[1, 2, ::3] = np.nan
    y[2] = np.nan
    y[1, 0, 7] = np.inf
    y[0, 3, [5, 9]] = np.inf
    _beam(y, s, zero, zero)
    t = s.copy()
    t[0, 2], t[1, 1], t[2] = np.nan, -np.inf, -np.inf
    _beam(x, t, zero, zero)
    _beam(x, s, zero, zero, (0, V), np.full(G, 1, np.int32))               # nothing allowed
    _beam(x, s, zero, zero, (0, V))                                        # everything ends
    few = np.full((G, K, V), -np.inf, np.float32)
    few[:, 1, 250], few[:, 3, 17] = 0.0, -1.0
    _beam(few, s, zero, zero)
    one = np.ones((G, K), np.int32)
    _beam(x, s, one * 5, one, (1, 4), None, 1.0)
    _beam(x, s, one * 0, one, (1, 4), None, 1.0)                           # finished without a token
    done = zero.copy()
    done[:, 2] = 1
    _beam(few, t, one * 3, done, (17, 18), np.full(G, 9, np.int32), 0.5)


def test_beam_close_keys_across_hypotheses():
    """Scores that differ by one fp32 step decide between hypotheses with equal logits."""
    rng = np.random.default_rng(1)
    G, K, V = 5, 8, 7000
    row = rng.normal(size=(G, 1, V)) * 2
    logits = np.repeat(row, K, 1).astype(np.float32)
    scores = np.full((G, K), -20.0, np.float32)
    for k in range(1, K):
        scores[:, k] = np.nextafter(scores[:, k - 1], np.float32(0 if k % 3 else -99))
    _beam(logits, scores, np.full((G, K), 9, np.int32), np.zeros((G, K), np.int32), None, None, 0.9)


def test_beam_in_place_and_strided():
    """State updated in its own buffers; logits that are rows of a wider buffer."""
    import torch
    ops = _ops()
    rng = np.random.default_rng(21)
    G, K, V = 4, 5, 1000
    scores, counts, done = _state(rng, G, K)
    sd, cd, dd = _cuda(scores), _cuda(counts), _cuda(done)
    out = ops.BeamStep(torch.empty(G, K, dtype=torch.int64, device="cuda"),
                       torch.empty(G, K, dtype=torch.int32, device="cuda"), sd, cd, dd)
    for _ in range(5):
        wide = rng.normal(size=(G, K, V + 24)).astype(np.float32)
        tok, par, scores, counts, done = ref.beam(wide[..., 8:8 + V], scores, counts, done, (990, 1000))
        scores = scores.astype(np.float32)
        done = done.astype(np.int32)
        ops.beam_select(_cuda(wide)[..., 8:8 + V], sd, cd, dd, stop=(990, 1000), out=out)
        assert np.array_equal(_np(out.tokens), tok) and np.array_equal(_np(out.parents), par)
        assert np.array_equal(_np(cd), counts) and np.array_equal(_np(dd), done)
        assert np.all(np.abs(_np(sd) - scores) <= 2.0 ** -23 * np.abs(scores))
        scores = _np(sd)


@pytest.mark.parametrize("K", [1, 2, 4, 5, 8, 11, 16, 32])
@pytest.mark.parametrize("ps,dim,cache", [(16, 64, "f32"), (1, 32, "f16"), (7, 96, "bf16"), (32, 128, "f32")])
@pytest.mark.parametrize("layers", [None, 3])
def test_reorder(K, ps, dim, cache, layers):
    ops = _ops()
    rng = np.random.default_rng(K * ps)
    G, kv, cols = 4, 2, 5
    lens = np.repeat(rng.integers(0, cols * ps + 1, G), K).astype(np.int32)
    lens[:K] = 0
    lens[-K:] = cols * ps
    if G > 2:
        lens[K:2 * K] = 2 * ps + max(ps // 2, 0)
    P = G * K * cols
    tables = rng.permutation(P).astype(np.int32).reshape(G * K, cols)
    parents = rng.integers(0, K, (G, K)).astype(np.int32)
    parents[0] = np.arange(K)
    if K > 2:
        parents[1] = np.roll(np.arange(K), 1)     # a cycle
        parents[2, 0], parents[2, 1] = -1, K      # outside: they stay
        tables[2 * K + 2, :] = [P, -1, P + 5, -9, P][:cols]   # a beam without pages of the pool
    L = layers or 1
    k, v = (_cuda(rng.normal(size=(L, P, kv, ps, dim)).astype(np.float32), _dt(cache)) for _ in range(2))
    wk, wv, wt = ref.reorder(_np(k), _np(v), tables, parents, lens)
    td = _cuda(tables)
    kk, vv = (k, v) if layers else (k[0], v[0])
    ops.paged_reorder(kk, vv, td, _cuda(parents), _cuda(lens))
    assert np.array_equal(_np(td), wt)
    assert np.array_equal(_np(k), wk) and np.array_equal(_np(v), wv)


# ---------------------------------------------------------------------------
# together, and in graphs
# ---------------------------------------------------------------------------

def test_chain_of_steps_equals_whole_sequences():
    """Requests that join, grow and leave through extend + append: after every step the paged
    attention of each request equals the plain attention over its whole history."""
    import torch
    ops = _ops()
    rng = np.random.default_rng(11)
    B, H, kv, D, ps, P, cols = 5, 6, 2, 64, 4, 60, 12
    k, v = torch.full((P, kv, ps, D), float("nan"), device="cuda"), torch.full((P, kv, ps, D), float("nan"), device="cuda")
    tables = torch.full((B, cols), -1, dtype=torch.int32, device="cuda")
    free, count = torch.arange(P, dtype=torch.int32, device="cuda"), torch.tensor([P], dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    hist = [np.zeros((0, 2 * kv, D), np.float32) for _ in range(B)]
    for step in range(14):
        new = rng.integers(0, 9, B) if step % 5 == 0 else np.ones(B, int)
        rel = (rng.random(B) < 0.15).astype(np.int32)
        T = 48
        qkv = rng.normal(size=(T, (H + 2 * kv) * D)).astype(np.float32)
        r = ops.paged_extend(lens, _cuda(new.astype(np.int32)), tables, free, count, ps, T, release=_cuda(rel))
        lens, count = r.lens, r.free_count
        q = ops.paged_append(_cuda(qkv), r.slots, r.pos, k, v, H)
        assert np.array_equal(_np(q).reshape(T, -1), qkv[:, :H * D])
        at = 0
        for b in range(B):
            hist[b] = np.concatenate([hist[b][:0] if rel[b] else hist[b],
                                      qkv[at:at + new[b]].reshape(-1, H + 2 * kv, D)[:, H:]])
            at += new[b]
        x = rng.normal(size=(B, H, D)).astype(np.float32)
        got = _np(ops.paged_attention(_cuda(x), k, v, tables, lens))
        for b in range(B):
            n = len(hist[b])
            assert int(lens[b]) == n
            one = hist[b].transpose(1, 0, 2)[:, None]          # a pool of one page holding all
            want, _ = ref.attention(x[b:b + 1], one[:kv].transpose(1, 0, 2, 3), one[kv:].transpose(1, 0, 2, 3),
                                    np.zeros((1, 1), np.int32), [n], D ** -0.5) if n else (np.zeros((1, H, D)), None)
            assert np.abs(got[b] - want[0]).max() <= 1e-5 * max(np.abs(want).max(), 1e-9)
    held = sum(-(-len(h) // ps) for h in hist)
    assert int(count) == P - held


def test_beams_follow_through_the_cache():
    """extend + append + reorder over beams: each beam's attention equals the one over the history of
    the hypothesis it stands for."""
    import torch
    ops = _ops()
    rng = np.random.default_rng(13)
    G, K, H, kv, D, ps, cols = 2, 4, 4, 2, 32, 3, 12
    B, P = G * K, G * K * 12
    k, v = (torch.zeros(2, P, kv, ps, D, device="cuda") for _ in range(2))
    tables = torch.full((B, cols), -1, dtype=torch.int32, device="cuda")
    free, count = torch.arange(P, dtype=torch.int32, device="cuda"), torch.tensor([P], dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    ones = torch.ones(B, dtype=torch.int32, device="cuda")
    hist = [np.zeros((2, 0, 2 * kv, D), np.float32) for _ in range(B)]
    for step in range(20):
        r = ops.paged_extend(lens, ones, tables, free, count, ps, B)
        lens, count = r.lens, r.free_count
        rows = rng.normal(size=(2, B, (H + 2 * kv) * D)).astype(np.float32)
        for layer in range(2):
            ops.paged_append(_cuda(rows[layer]), r.slots, r.pos, k[layer], v[layer], H)
        hist = [np.concatenate([hist[b], rows[:, b].reshape(2, 1, H + 2 * kv, D)[:, :, H:]], 1) for b in range(B)]
        x = rng.normal(size=(B, H, D)).astype(np.float32)
        for layer in range(2):
            got = _np(ops.paged_attention(_cuda(x), k[layer], v[layer], tables, lens))
            for b in range(B):
                one = hist[b][layer].transpose(1, 0, 2)
                want, _ = ref.attention(x[b:b + 1], one[None, :kv], one[None, kv:], np.zeros((1, 1), np.int32), [step + 1],
                                        D ** -0.5)
                assert np.abs(got[b] - want[0]).max() <= 1e-5 * np.abs(want).max(), (step, layer, b)
        par = rng.integers(0, K, (G, K)).astype(np.int32)
        ops.paged_reorder(k, v, tables, _cuda(par), lens)
        hist = [hist[g * K + par[g, i]] for g in range(G) for i in range(K)]


def test_graph_replay_on_a_side_stream():
    """A step captured once on a side stream and replayed with changed lengths and inputs, next to a
    second captured graph of the same call, equals eager calls."""
    import torch
    ops = _ops()
    rng = np.random.default_rng(17)
    B, H, kv, D, ps, cols = 3, 14, 2, 64, 16, 80
    P = B * cols
    tables = _cuda(rng.permutation(P).astype(np.int32).reshape(B, cols))
    k, v = (_cuda(rng.normal(size=(P, kv, ps, D)).astype(np.float32)) for _ in range(2))
    graphs = []
    for i in range(2):
        q = torch.zeros(B, H, D, device="cuda")
        lens = torch.ones(B, dtype=torch.int32, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = ops.paged_attention(q, k, v, tables, lens)
        graphs.append((g, q, lens, out))
    for trial in range(4):
        feeds = [(_cuda(rng.normal(size=(B, H, D)).astype(np.float32)),
                  _cuda(rng.integers(0, cols * ps + 1, B).astype(np.int32))) for _ in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        for (g, q, lens, out), (fq, fl), s in zip(graphs, feeds, streams):
            q.copy_(fq)
            lens.copy_(fl)
        torch.cuda.synchronize()
        for (g, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (g, q, lens, out), (fq, fl) in zip(graphs, feeds):
            assert torch.equal(out, ops.paged_attention(fq, k, v, tables, fl))


# ---------------------------------------------------------------------------
# the two ways of a call
# ---------------------------------------------------------------------------

def test_short_and_long_way_agree(monkeypatch):
    """The extension module takes the plain calls and gives what the Python way gives, bit for bit; the
    calls it does not take are refused with the Python way's messages."""
    import torch
    ops, P = _ops(), pkg("paged")
    mod = P._bind()
    assert mod, "the extension module was not built"
    rng = np.random.default_rng(31)
    tables, Pn, rest = _tables(rng, [40, 0, 333], 16, 24)
    stack = np.zeros(Pn, np.int32)
    stack[:len(rest)] = rest
    k, v = (_cuda(rng.normal(size=(2, Pn, 2, 16, 64)).astype(np.float32)) for _ in range(2))
    lens, new = _cuda(np.array([40, 0, 333], np.int32)), _cuda(np.array([1, 1, 1], np.int32))
    qkv = _cuda(rng.normal(size=(3, 18 * 64)).astype(np.float32))
    tab = _cuda(rng.normal(size=(400, 64)).astype(np.float32))
    logits = _cuda(rng.normal(size=(1, 3, 777)).astype(np.float32))
    scores, z = _cuda(rng.normal(size=(1, 3)).astype(np.float32)), torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")

    def all_of_them():
        kk, vv, td, sd = k.clone(), v.clone(), _cuda(tables), _cuda(stack)
        cd = _cuda(np.array([len(rest)], np.int32))
        r = ops.paged_extend(lens, new, td, sd, cd, 16, 4, release=_cuda(np.array([0, 1, 0], np.int32)))
        q = ops.paged_append(qkv, r.slots[:3], r.pos[:3], kk[1], vv[1], 14, tab, tab, bad=bad)
        q2 = ops.paged_append(qkv, r.slots[:3], None, kk[0], vv[0], 14, out=torch.empty_like(q))
        o, lse = ops.paged_attention(q, kk[1], vv[1], td, r.lens, scale=0.2, window=100, return_lse=True, bad=bad)
        o2 = ops.paged_attention(q, kk[1], vv[1], td, r.lens)
        b = ops.beam_select(logits, scores, z, z, stop=(700, 777), length_penalty=0.5)
        ops.paged_reorder(kk, vv, td, b.parents, r.lens)
        ops.paged_reorder(kk[0], vv[0], td, b.parents, r.lens)
        assert type(r) is ops.PagedStep and type(b) is ops.BeamStep
        return [*r, q, q2, o, lse, o2, *b, kk, vv, td, sd]

    taken = []
    for name in ("extend", "append", "attention", "beam", "reorder"):
        def spy(*a, f=getattr(mod, name), name=name):
            r = f(*a)
            taken.append((name, r is not None))
            return r
        monkeypatch.setattr(mod, name, spy)
    short = all_of_them()
    assert len(taken) == 8 and all(t for _, t in taken)
    monkeypatch.setattr(P, "_bound", False)
    monkeypatch.setattr(P, "_bind", lambda: False)
    for a, b in zip(short, all_of_them()):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def test_refusals_on_the_device():
    import torch
    ops = _ops()
    k = torch.zeros(3, 2, 16, 64, device="cuda")
    q = torch.zeros(2, 4, 64, device="cuda")
    t, n = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    ops.paged_attention(q, k, k, t, n)
    for a in ((q.cpu(), k, k, t, n), (q, k.cpu(), k, t, n), (q, k, k, t, n.long()), (q[:, :3], k, k, t, n), (q, k, k, t.T, n),
              (q, k, k.half(), t, n), (q.double(), k, k, t, n), (q, k[..., :32], k[..., :32], t, n)):
        with pytest.raises(ValueError):
            ops.paged_attention(*a)
    with pytest.raises(ValueError):
        ops.paged_attention(q, k, k, t, n, window=-1)
    with pytest.raises(ValueError):
        ops.paged_attention(q, k.view(3, 2, 16, 64)[..., 1:], k[..., 1:], t, n)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.paged_attention(torch.zeros(2, 4, 80, device="cuda"), torch.zeros(3, 2, 16, 80, device="cuda"),
                            torch.zeros(3, 2, 16, 80, device="cuda"), t, n)
    off = torch.zeros(3 * 2 * 16 * 64 + 4, device="cuda")[4:].view(3, 2, 16, 64)
    with pytest.raises(ValueError, match="32-byte"):
        ops.paged_attention(q, off, off, t, n)
    with pytest.raises(RuntimeError, match="beams"):
        ops.beam_select(torch.zeros(1, 33, 9, device="cuda"), torch.zeros(1, 33, device="cuda"),
                        *(torch.zeros(1, 33, dtype=torch.int32, device="cuda") for _ in range(2)))
    with pytest.raises(ValueError):
        ops.beam_select(torch.zeros(1, 3, 9, device="cuda"), torch.zeros(1, 3, device="cuda"),
                        *(torch.zeros(1, 3, dtype=torch.int32, device="cuda") for _ in range(2)), stop=(0, 10))


def test_numpy_host():
    """The operators on the library's own device arrays, PyTorch blocked: the chain's results equal the
    64-bit restatement's (tolerances as above)."""
    import subprocess
    import sys
    from conftest import REPO
    child = r"""
import importlib, sys
sys.modules["torch"] = None
sys.path.insert(0, sys.argv[1])
import numpy as np
import oracle.paged as ref
P = "cosyvoice3-cpu_b200."
ops, D = importlib.import_module(P + "ops"), importlib.import_module(P + "_dev")
assert D.BACKEND == "numpy"
up = D.DeviceArray.from_numpy
rng = np.random.default_rng(0)
B, H, Hk, d, ps, cols, pages = 3, 6, 2, 64, 16, 6, 24
k, v = np.zeros((2, pages, Hk, ps, d), np.float32), np.zeros((2, pages, Hk, ps, d), np.float32)
tables, stack = np.full((B, cols), -1, np.int32), np.arange(pages, dtype=np.int32)
lens, new = np.zeros(B, np.int32), np.array([40, 0, 90], np.int32)
kd, vd, td, sd = up(k), up(v), up(tables), up(stack)
r = ops.paged_extend(up(lens), up(new), td, sd, up(np.array([pages], np.int32)), ps, 131)
tables, stack, slots, seq, pos, offsets, lens, count = ref.extend(lens, new, tables, stack, pages, ps, 131)
for a, b in zip(r, (slots, seq, pos, offsets, lens, np.array([count], np.int32))):
    assert np.array_equal(a.numpy(), b)
qkv = rng.normal(size=(131, (H + 2 * Hk) * d)).astype(np.float32)
cos, sin = rng.normal(size=(2, 100, d)).astype(np.float32)
q = ops.paged_append(up(qkv), r.slots, r.pos, kd[1], vd[1], H, up(cos), up(sin))
x = qkv.reshape(131, H + 2 * Hk, d)
turned = ref.rope_rows(x[:, :H + Hk], cos[pos], sin[pos])
assert np.abs(q.numpy() - turned[:, :H]).max() < 3e-6
k[1][slots[:130] // ps, :, slots[:130] % ps] = turned[:130, H:]
v[1][slots[:130] // ps, :, slots[:130] % ps] = x[:130, H + Hk:]
assert np.abs(kd.numpy() - k).max() < 3e-6 and np.array_equal(vd.numpy(), v)
qq = rng.normal(size=(B, H, d)).astype(np.float32)
o, lse = ops.paged_attention(up(qq), kd[1], vd[1], td, r.lens, return_lse=True)
want, wl = ref.attention(qq, kd.numpy()[1], v[1], tables, lens, d ** -0.5)
assert np.abs(o.numpy() - want).max() < 1e-5 * np.abs(want).max() and not o.numpy()[1].any()
logits = rng.normal(size=(1, 3, 500)).astype(np.float32)
s, z = rng.normal(size=(1, 3)).astype(np.float32), np.zeros((1, 3), np.int32)
b = ops.beam_select(up(logits), up(s), up(z), up(z), stop=(490, 500))
w = ref.beam(logits, s, z, z, (490, 500))
assert np.array_equal(b.tokens.numpy(), w[0]) and np.array_equal(b.parents.numpy(), w[1])
par = np.array([[2, 0, 0]], np.int32)
n = np.full(3, 21, np.int32)
t3 = np.arange(18, dtype=np.int32).reshape(3, 6)
t3d = up(t3)
kk, vv = kd.numpy(), vd.numpy()
ops.paged_reorder(kd, vd, t3d, up(par), up(n))
wk, wv, wt = ref.reorder(kk, vv, t3, par, n)
assert np.array_equal(kd.numpy(), wk) and np.array_equal(vd.numpy(), wv) and np.array_equal(t3d.numpy(), wt)
try:
    ops.paged_attention(qq, kd[1], vd[1], td, r.lens)
except ValueError:
    print("numpy host ok")
"""
    r = subprocess.run([sys.executable, "-c", child, REPO], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "numpy host ok" in r.stdout, r.stderr[-2000:]
