"""Pages that several table rows name: counted, given back once, against the oracle's restatement (whole numbers,
exact), and what requests read afterwards."""

import numpy as np
import pytest

from conftest import pkg

import oracle.paged as ref

pytestmark = pytest.mark.gpu


def _cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _shared_tables(rng, rows, cols, ps):
    """Rows in groups of 1 to 5 that share a prefix of pages: (tables, lens, pages, shares, free pages)."""
    lens = rng.integers(0, cols * ps + 1, rows).astype(np.int32)
    tables, used = np.full((rows, cols), -1, np.int32), 0
    b = 0
    while b < rows:
        n = min(int(rng.integers(1, 6)), rows - b)
        held = -(-lens[b:b + n] // ps)
        common = int(rng.integers(0, held.min() + 1))
        tables[b:b + n, :common] = np.arange(used, used + common)
        used += common
        for r in range(b, b + n):
            tables[r, common:held[r - b]] = np.arange(used, used + held[r - b] - common)
            used += held[r - b] - common
        b += n
    P = used + rows + 7
    ids = rng.permutation(P).astype(np.int32)
    tables = np.where(tables >= 0, ids[tables], -1).astype(np.int32)
    shares = np.zeros(P, np.int32)
    named = np.bincount(tables[tables >= 0], minlength=P)
    shares[:] = np.maximum(named - 1, 0)
    return tables, lens, P, shares, ids[used:]


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 40, 600, 1500, 9000])
@pytest.mark.parametrize("ps,cols", [(1, 70), (7, 5), (16, 33)])
@pytest.mark.parametrize("part", [0.3, 1.0])
def test_extend_releases_shared_pages_once(rows, ps, cols, part):
    ops = pkg("ops")
    rng = np.random.default_rng(rows + ps)
    tables, lens, P, shares, rest = _shared_tables(rng, rows, cols, ps)
    stack = np.full(P, -7, np.int32)
    stack[:len(rest)] = rest
    release = (rng.random(rows) < part).astype(np.int32) * 3
    if rows > 20:
        tables[3, 0], tables[9, 1] = P, -5          # page numbers outside the pool are passed over
    new = np.where(release, rng.integers(0, cols * ps + 1, rows), rng.integers(0, 2, rows)).astype(np.int32)
    T = int(new.sum()) + 3
    s2, count, sh2, held = ref.give_back(tables, lens, ps, stack, len(rest), shares, release=release)
    want = ref.extend(held, new, tables, s2, count, ps, T)
    td, sd, ld, cd, shd = _cuda(tables), _cuda(stack), _cuda(lens), _cuda(np.array([len(rest)], np.int32)), _cuda(shares)
    got = ops.paged_extend(ld, _cuda(new), td, sd, cd, ps, T, release=_cuda(release), shares=shd)
    assert np.array_equal(td.cpu().numpy(), want[0]) and np.array_equal(shd.cpu().numpy(), sh2)
    assert int(got.free_count) == want[7] and np.array_equal(sd.cpu().numpy()[:count], want[1][:count])
    for a, b in zip((got.slots, got.seq, got.pos, got.offsets, got.lens), want[2:7]):
        assert np.array_equal(a.cpu().numpy(), b)
    assert np.array_equal(ld.cpu().numpy(), lens) and int(cd) == len(rest)      # the inputs stay
    # in place, and without any release
    step = ops.PagedStep(*got[:4], ld, cd)
    td, sd, shd = _cuda(tables), _cuda(stack), _cuda(shares)
    ops.paged_extend(ld, _cuda(new), td, sd, cd, ps, T, release=_cuda(release), out=step, shares=shd)
    assert np.array_equal(ld.cpu().numpy(), want[6]) and int(cd) == want[7] and np.array_equal(shd.cpu().numpy(), sh2)
    ops.paged_extend(ld, _cuda(new * 0), td, sd, cd, ps, T, out=step, shares=shd)
    assert np.array_equal(shd.cpu().numpy(), sh2) and int(cd) == want[7]


def test_rows_left_uncounted_go_back_once():
    """Rows that share pages nobody counted, released in one call: still one time each."""
    ops = pkg("ops")
    tables = np.array([[0, 1], [0, 1], [0, 2]], np.int32)
    i32 = lambda *x: _cuda(np.array(x, np.int32))  # noqa: E731
    stack, shares = i32(-1, -1, -1, -1), i32(0, 0, 0, 0)
    r = ops.paged_extend(i32(8, 8, 8), i32(0, 0, 0), _cuda(tables), stack, i32(0), 4, 0, release=i32(1, 1, 1), shares=shares)
    assert int(r.free_count) == 3 and stack.tolist() == [0, 1, 2, -1] and shares.tolist() == [0] * 4


@pytest.mark.parametrize("K", [1, 2, 5, 8, 32])
@pytest.mark.parametrize("G", [1, 3, 40])
@pytest.mark.parametrize("ps", [1, 4])
def test_reorder_counts_and_gives_back(K, G, ps):
    """A walk of growth and choices: tables, counts and the stack follow the restatement, every page is on the
    stack or named, and the counts are those of the tables."""
    ops = pkg("ops")
    rng = np.random.default_rng(K * 100 + G)
    cols, B = 9, G * K
    P = B * cols + 5
    k, v = (_cuda(rng.normal(size=(2, P, 1, ps, 8)).astype(np.float32)) for _ in range(2))
    tables, stack, count = np.full((B, cols), -1, np.int32), rng.permutation(P).astype(np.int32), P
    lens, shares = np.zeros(B, np.int32), np.zeros(P, np.int32)
    td, sd, cd, shd = _cuda(tables), _cuda(stack), _cuda(np.array([P], np.int32)), _cuda(shares)
    ld = _cuda(lens)
    for step in range(7):
        new = np.repeat(rng.integers(0, ps + 1, G), K).astype(np.int32)
        release = None
        if step in (3, 5):
            release = np.repeat(rng.random(G) < 0.4, K).astype(np.int32)
            stack, count, shares, lens = ref.give_back(tables, lens, ps, stack, count, shares, release=release)
            release = _cuda(release)
        T = int(new.sum())
        tables, stack, *_, lens, count = ref.extend(lens, new, tables, stack, count, ps, T)
        r = ops.paged_extend(ld, _cuda(new), td, sd, cd, ps, T, release=release, shares=shd)
        ld, cd = r.lens, r.free_count
        parents = rng.integers(-1, K + 1, (G, K)).astype(np.int32)
        stack, count, shares, _ = ref.give_back(tables, lens, ps, stack, count, shares, parents=parents)
        wk, wv, tables = ref.reorder(k.cpu().numpy(), v.cpu().numpy(), tables, parents, lens)
        ops.paged_reorder(k, v, td, _cuda(parents), ld, shd, sd, cd)
        assert np.array_equal(td.cpu().numpy(), tables) and np.array_equal(shd.cpu().numpy(), shares)
        assert int(cd) == count and np.array_equal(sd.cpu().numpy()[:count], stack[:count])
        assert np.array_equal(k.cpu().numpy(), wk) and np.array_equal(v.cpu().numpy(), wv)
        named = np.bincount(np.concatenate([tables[b, :-(-int(lens[b]) // ps)] for b in range(B)]), minlength=P)
        free = np.bincount(stack[:count], minlength=P)
        assert np.array_equal(free, (named == 0).astype(free.dtype)) and np.array_equal(shares, np.maximum(named - 1, 0))


def test_released_beams_leave_room_for_prompts_of_their_own():
    """Beams that follow one parent are released; the prompts that take their places share no page and no slot,
    and each reads back what it wrote."""
    import torch
    ops = pkg("ops")
    cache = pkg("models.paged").PagedKVCache(1, 2, 64, requests=2, max_len=32, pages=4, page_size=16)
    i32 = dict(dtype=torch.int32, device="cuda")
    cache.extend(torch.tensor([32, 32], **i32), 64)
    cache.reorder(torch.tensor([[0, 0]], **i32))
    assert int(cache.free_count) == 2 and torch.equal(cache.tables[0], cache.tables[1])
    step = cache.extend(torch.tensor([32, 32], **i32), 64, release=torch.tensor([1, 1], **i32))
    assert sorted(cache.tables.view(-1).tolist()) == [0, 1, 2, 3] and int(cache.free_count) == 0
    assert len(set(step.slots.tolist())) == 64 and not bool(cache.shares.any())
    rng = np.random.default_rng(0)
    qkv = _cuda(rng.normal(size=(64, 6 * 64)).astype(np.float32))
    ops.paged_append(qkv, step.slots, None, cache.k[0], cache.v[0], 2, bad=cache.bad)
    q = _cuda(rng.normal(size=(2, 2, 64)).astype(np.float32))
    got = cache.attention(0, q, 0.125).cpu().numpy()
    x = qkv.view(2, 32, 6, 64).cpu().numpy()
    for b in range(2):
        one = x[b].transpose(1, 0, 2)[None]
        want, _ = ref.attention(q[b:b + 1].cpu().numpy(), one[:, 2:4], one[:, 4:], np.zeros((1, 1), np.int32), [32], 0.125)
        # fp32 attention, tolerance as in the suite's other tests of it
        assert np.abs(got[b] - want[0]).max() <= 1e-5 * np.abs(want).max()
    assert int(cache.bad) == 0


def test_beams_of_a_prefill_are_released():
    """The pages that start_beams shares come back one time; a cache that counts none refuses releases."""
    import torch
    P = pkg("models.paged")
    c = pkg("models.qwen2").KVCache(1, 2, 64, 2, 64)
    for t in (c.k, c.v):
        t.normal_()
    cache = P.PagedKVCache(1, 2, 64, requests=6, max_len=64, pages=30, page_size=16)
    cache.start_beams([37, 16], c, 3)
    i32 = dict(dtype=torch.int32, device="cuda")
    assert cache.shares.tolist() == [2, 2, 0, 0, 0, 2] + [0] * 24 and int(cache.free_count) == 24
    assert torch.equal(cache.k[0, 5], c.k[0, 1, :, :16]) and torch.equal(cache.k[0, 4, :, :5], c.k[0, 0, :, 32:37])
    zero = torch.zeros(6, **i32)
    cache.extend(zero, 0, release=torch.tensor([1, 1, 0, 0, 0, 0], **i32))
    assert int(cache.free_count) == 26 and cache.shares.tolist() == [0, 0, 0, 0, 0, 2] + [0] * 24
    cache.extend(zero, 0, release=torch.tensor([0, 0, 1, 1, 1, 1], **i32))
    assert int(cache.free_count) == 30 and sorted(cache.free.tolist()) == list(range(30)) and not bool(cache.shares.any())
    plain = P.PagedKVCache(1, 2, 64, requests=2, max_len=64, pages=30, page_size=16, releases=False)
    plain.extend(torch.ones(2, **i32), 2)
    plain.reorder(torch.zeros(1, 2, **i32))
    with pytest.raises(ValueError, match="releases=False"):
        plain.extend(torch.ones(2, **i32), 2, release=torch.ones(2, **i32))


def test_shared_pages_in_a_captured_step():
    """A captured step with releases and choices, replayed, does what eager calls do."""
    import torch
    ops = pkg("ops")
    rng = np.random.default_rng(2)
    G, K, ps, cols = 20, 4, 2, 6
    B, P, T = G * K, G * K * cols, 2 * G * K
    pool = torch.zeros(1, P, 1, ps, 8, device="cuda")

    def state():
        i32 = dict(dtype=torch.int32, device="cuda")
        return dict(lens=torch.zeros(B, **i32), tables=torch.full((B, cols), -1, **i32), free=torch.arange(P, **i32),
                    count=torch.full((1,), P, **i32), shares=torch.zeros(P, **i32), new=torch.zeros(B, **i32),
                    release=torch.zeros(B, **i32), parents=torch.zeros(G, K, **i32),
                    out=[torch.zeros(T, dtype=torch.int64, device="cuda")] + [torch.zeros(n, **i32) for n in (T, T, B + 1)])

    def step(s):
        ops.paged_extend(s["lens"], s["new"], s["tables"], s["free"], s["count"], ps, T, release=s["release"],
                         out=ops.PagedStep(*s["out"], s["lens"], s["count"]), shares=s["shares"])
        ops.paged_reorder(pool, pool.clone(), s["tables"], s["parents"], s["lens"], s["shares"], s["free"], s["count"])
    a, b = state(), state()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        step(b)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(6):
        new = np.repeat(rng.integers(0, 3, G), K).astype(np.int32)
        rel = np.repeat(rng.random(G) < 0.3, K).astype(np.int32)
        par = rng.integers(0, K, (G, K)).astype(np.int32)
        for s in (a, b):
            for name, x in (("new", new), ("release", rel), ("parents", par)):
                s[name].copy_(torch.from_numpy(x))
        step(a)
        g.replay()
        n = int(a["count"])
        assert n == int(b["count"]) and torch.equal(a["free"][:n], b["free"][:n])
        for name in ("lens", "tables", "shares"):
            assert torch.equal(a[name], b[name]), name


def test_shared_pages_on_the_numpy_host():
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
up = D.DeviceArray.from_numpy
tables, lens = np.array([[0, 1], [2, 3], [4, 5]], np.int32), np.full(3, 8, np.int32)
stack, shares, par = np.full(6, -1, np.int32), np.zeros(6, np.int32), np.array([[2, 2, 2]], np.int32)
pool = np.zeros((6, 1, 4, 8), np.float32)
td, sd, shd, cd = up(tables), up(stack), up(shares), up(np.zeros(1, np.int32))
ops.paged_reorder(up(pool), up(pool), td, up(par), up(lens), shd, sd, cd)
assert sd.numpy().tolist() == [0, 1, 2, 3, -1, -1] and shd.numpy().tolist() == [0, 0, 0, 0, 2, 2] and cd.numpy()[0] == 4
new = up(np.array([1, 0, 1], np.int32))
r = ops.paged_extend(up(lens), new, td, sd, cd, 4, 3, release=up(np.array([1, 0, 1], np.int32)), shares=shd)
assert r.free_count.numpy()[0] == 2 and shd.numpy().tolist() == [0] * 6 and r.lens.numpy().tolist() == [1, 8, 1]
assert td.numpy().tolist() == [[3, 5], [4, 5], [2, 5]]
print("numpy host ok")
"""
    r = subprocess.run([sys.executable, "-c", child, REPO], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "numpy host ok" in r.stdout, r.stderr[-2000:]


def test_no_requests_and_no_groups():
    """Empty batches are fine with counts as without."""
    import torch
    ops = pkg("ops")
    i32 = dict(dtype=torch.int32, device="cuda")
    e, t, s, c = torch.zeros(0, **i32), torch.zeros(0, 3, **i32), torch.arange(4, **i32), torch.full((1,), 3, **i32)
    sh = torch.zeros(4, **i32)
    r = ops.paged_extend(e, e, t, s, c, 16, 2, release=e, shares=sh)
    assert int(r.free_count) == 3 and r.slots.tolist() == [-1, -1] and r.offsets.tolist() == [0]
    k = torch.zeros(4, 1, 16, 8, device="cuda")
    ops.paged_reorder(k, k, t, torch.zeros(0, 4, **i32), e, sh, s, c)
    one = torch.zeros(1, 3, **i32)
    ops.paged_reorder(k, k, one, torch.zeros(1, 1, **i32), torch.full((1,), 33, **i32), sh, s, c)
    assert int(c) == 3 and not bool(sh.any()) and s.tolist() == [0, 1, 2, 3]
