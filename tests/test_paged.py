"""Refusals of the paged-cache and beam-search operators, without a GPU: host arrays, shapes, types,
strides and alignment are rejected before anything reaches the device (the host checks run here on
CPU tensors with the device check replaced, the C ABI on made-up addresses that it must not touch)."""

import os
import re

import numpy as np
import pytest

from conftest import REPO, pkg

import oracle.paged as ref


@pytest.fixture
def ops(monkeypatch):
    import torch
    p = pkg("paged")
    monkeypatch.setattr(p, "_device", lambda name, *arrays: 0)

    def no_launch():
        raise AssertionError("the arguments were accepted")
    monkeypatch.setattr(p, "load", no_launch)
    monkeypatch.setattr(p.D, "require_cuda", lambda: None)
    monkeypatch.setattr(p.D, "empty", lambda shape, dtype=None: torch.empty(shape, dtype=dtype or torch.float32))
    return p


def _i32(*shape):
    import torch
    return torch.zeros(shape, dtype=torch.int32)


def test_host_arrays_are_refused():
    import torch
    p = pkg("paged")
    x = torch.zeros(2, 4, 64)
    pool = torch.zeros(3, 2, 16, 64)
    for bad in (x, x.numpy()):
        with pytest.raises(ValueError, match="CUDA tensors are expected"):
            p.paged_attention(bad, pool, pool, _i32(2, 3), _i32(2))
    with pytest.raises(ValueError, match="CUDA tensors are expected"):
        p.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2), _i32(1, 2), _i32(1, 2))
    with pytest.raises(ValueError, match="CUDA tensors are expected"):
        p.paged_extend(_i32(2), _i32(2), _i32(2, 3), _i32(9), _i32(1), 16, 4)
    with pytest.raises(ValueError, match="CUDA tensors are expected"):
        p.paged_append(torch.zeros(2, 8 * 64), torch.zeros(2, dtype=torch.int64), _i32(2), pool, pool, 4)
    with pytest.raises(ValueError, match="CUDA tensors are expected"):
        p.paged_reorder(pool, pool, _i32(4, 3), _i32(2, 2), _i32(4))


def test_other_devices_are_refused(monkeypatch):
    import torch
    p = pkg("paged")

    class On:
        def __init__(self, d):
            self.d = d

        def get_device(self):
            return self.d
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    assert p._device("op", On(0), On(0)) == 0
    with pytest.raises(ValueError, match="cuda:0 and cuda:1"):
        p._device("op", On(0), On(1))
    with pytest.raises(ValueError, match="current device is cuda:0"):
        p._device("op", On(1), On(1))


def test_extend_refusals(ops):
    import torch
    good = dict(lens=_i32(3), new_lens=_i32(3), block_tables=_i32(3, 5), free_pages=_i32(9), free_count=_i32(1),
                page_size=16, max_tokens=4)
    with pytest.raises(AssertionError, match="accepted"):
        ops.paged_extend(**good)
    for change in (dict(new_lens=_i32(2)), dict(lens=torch.zeros(3, dtype=torch.int64)), dict(block_tables=_i32(2, 5)),
                   dict(block_tables=_i32(5, 3).T), dict(free_count=_i32(2)), dict(page_size=0), dict(max_tokens=-1),
                   dict(release=_i32(4)), dict(lens=_i32(6)[::2]), dict(free_pages=torch.zeros(9)),
                   dict(out=ops.PagedStep(*[_i32(4)] * 6)), dict(lens=torch.tensor(3, dtype=torch.int32)),
                   dict(block_tables=torch.zeros(3, 5))):
        with pytest.raises(ValueError):
            ops.paged_extend(**{**good, **change})


def test_append_refusals(ops):
    import torch
    pool = torch.zeros(3, 2, 16, 64)
    tab = torch.zeros(50, 64)
    good = dict(qkv=torch.zeros(4, 8 * 64), slots=torch.zeros(4, dtype=torch.int64), pos=_i32(4), k_pages=pool,
                v_pages=pool.clone(), heads=4, cos=tab, sin=tab)
    with pytest.raises(AssertionError, match="accepted"):
        ops.paged_append(**good)
    for change in (dict(heads=5), dict(heads=0), dict(slots=_i32(4)), dict(slots=torch.zeros(3, dtype=torch.int64)),
                   dict(cos=None), dict(pos=None), dict(pos=_i32(5)), dict(cos=torch.zeros(50, 32)),
                   dict(cos=tab.double()), dict(k_pages=pool.double(), v_pages=pool.double()),
                   dict(v_pages=pool.half()), dict(v_pages=pool[:2]), dict(k_pages=pool[0], v_pages=pool[0]),
                   dict(k_pages=pool.transpose(2, 3), v_pages=pool.transpose(2, 3)),
                   dict(qkv=torch.zeros(4, 8 * 64, dtype=torch.int32)), dict(qkv=torch.zeros(8 * 64, 4).T),
                   dict(out=torch.zeros(4, 4, 32)), dict(bad=_i32(2)), dict(qkv=torch.zeros(4, 8, 64)),
                   dict(k_pages=pool[:1].expand(3, 2, 16, 64))):
        with pytest.raises(ValueError):
            ops.paged_append(**{**good, **change})


def test_attention_refusals(ops):
    import torch
    pool = torch.zeros(3, 2, 16, 64)
    good = dict(q=torch.zeros(2, 4, 64), k_pages=pool, v_pages=pool, block_tables=_i32(2, 3), lens=_i32(2))
    with pytest.raises(AssertionError, match="accepted"):
        ops.paged_attention(**good)
    for change in (dict(q=torch.zeros(2, 3, 64)), dict(q=torch.zeros(2, 4, 32)), dict(q=torch.zeros(4, 64)),
                   dict(q=torch.zeros(2, 64, 4).transpose(1, 2)), dict(q=torch.zeros(2, 4, 64, dtype=torch.float64)),
                   dict(lens=_i32(3)), dict(lens=torch.zeros(2)), dict(block_tables=_i32(3, 3)), dict(window=-1),
                   dict(out=torch.zeros(2, 4, 64, dtype=torch.float16)), dict(out=torch.zeros(4, 2, 64).transpose(0, 1)),
                   dict(v_pages=torch.zeros(3, 2, 8, 64)), dict(q=torch.zeros(2, 0, 64)), dict(bad=_i32(0)),
                   dict(k_pages=torch.zeros(3, 2, 0, 64), v_pages=torch.zeros(3, 2, 0, 64))):
        with pytest.raises(ValueError):
            ops.paged_attention(**{**good, **change})


def test_beam_and_reorder_refusals(ops):
    import torch
    good = dict(logits=torch.zeros(2, 3, 50), scores=torch.zeros(2, 3), counts=_i32(2, 3), done=_i32(2, 3))
    with pytest.raises(AssertionError, match="accepted"):
        ops.beam_select(**good)
    for change in (dict(logits=torch.zeros(6, 50)), dict(scores=torch.zeros(2, 2)), dict(scores=_i32(2, 3)),
                   dict(counts=torch.zeros(2, 3)), dict(done=torch.zeros(2, 3, dtype=torch.bool)), dict(stop=(3, 51)),
                   dict(stop=(5, 4)), dict(stop=(-1, 4)), dict(min_len=_i32(3)),
                   dict(logits=torch.zeros(2, 50, 3).transpose(1, 2)), dict(logits=torch.zeros(3, 2, 50).transpose(0, 1)),
                   dict(logits=torch.zeros(2, 3, 50, dtype=torch.int32)), dict(out=ops.BeamStep(*[_i32(2, 3)] * 5))):
        with pytest.raises(ValueError):
            ops.beam_select(**{**good, **change})
    pool = torch.zeros(2, 9, 2, 16, 64)
    fine = dict(k_pages=pool, v_pages=pool, block_tables=_i32(6, 3), parents=_i32(2, 3), lens=_i32(6))
    with pytest.raises(AssertionError, match="accepted"):
        ops.paged_reorder(**fine)
    for change in (dict(k_pages=pool[0, 0]), dict(v_pages=pool[0]), dict(block_tables=_i32(5, 3)), dict(parents=_i32(6)),
                   dict(lens=_i32(2)), dict(parents=torch.zeros(2, 3)), dict(k_pages=pool.int(), v_pages=pool.int()),
                   dict(v_pages=pool[:1].expand(2, 9, 2, 16, 64))):
        with pytest.raises(ValueError):
            ops.paged_reorder(**{**fine, **change})


BLOCKS = {"cv3_paged_extend": "_EXTEND", "cv3_paged_append": "_APPEND", "cv3_paged_attention": "_ATTENTION",
          "cv3_beam": "_BEAM", "cv3_paged_reorder": "_REORDER"}


def test_parameter_blocks_match_the_header():
    """Every field of a block is 8 bytes, doubles last: the packed format has the header's fields."""
    text = open(os.path.join(REPO, "include", "cv3cuda.h")).read()
    p = pkg("paged")
    for name, fmt in BLOCKS.items():
        body = re.search(r"typedef struct %s_params \{(.*?)\} %s_params;" % (name, name), text, re.S).group(1)
        kinds = []
        for line in filter(None, (x.strip() for x in body.split(";"))):
            t = "q" if "*" in line or line.startswith("int64_t") else "d" if line.startswith("double") else "?"
            kinds += [t] * len(line.split(","))
        f = getattr(p, fmt)
        assert "?" not in kinds and kinds == sorted(kinds, reverse=True)
        assert f.size == 8 * len(kinds) and f.unpack(f.pack(*([0] * len(kinds)))).count(0.0) == len(kinds)
        assert f.format.lstrip("=") in ("%dq" % len(kinds), "%dqd" % (len(kinds) - 1))
        assert f.format.endswith("d") == (kinds[-1] == "d")


def test_c_entries_refuse_before_any_device_work():
    L, p = pkg("_lib"), pkg("paged")
    lib = L.load()
    V, U = L.CV3_ERR_VALUE, L.CV3_ERR_UNSUPPORTED
    at = 1 << 20

    def attention(dim=64, kv=2, heads=4, ps=16, strides=(2048, 1024, 64), k=at, kt=0, cols=3, ld=3, window=0, batch=0,
                  words=0, size=p._ATTENTION.size):
        return lib.cv3_paged_attention(p._ATTENTION.pack(
            size, at, 0, heads * dim, dim, k, at, kt, *strides, *strides, 9, ps, at, ld, cols, at, batch, heads, kv, dim,
            window, at, heads * dim, dim, 0, 0, 0, words, 0.1), None)
    assert attention() == 0                                  # no requests: nothing to do
    assert attention(size=8) == V and b"parameter block" in lib.cv3_last_error()
    assert attention(dim=80) == U and b"head_dim" in lib.cv3_last_error()
    assert attention(kv=3) == V and b"not a multiple" in lib.cv3_last_error()
    assert attention(strides=(2048, 1024, 62)) == V and b"32-byte" in lib.cv3_last_error()
    assert attention(k=at + 16) == V
    assert attention(kt=5) == V and attention(ps=0) == V and attention(ld=2) == V and attention(window=-1) == V
    assert attention(cols=1 << 28, ld=1 << 28) == V and b"32-bit" in lib.cv3_last_error()
    assert attention(cols=5000, ld=5000, batch=2) == V and b"workspace" in lib.cv3_last_error()
    assert lib.cv3_paged_attention(None, None) == V

    def append(dim=64, ldq=8 * 64, rows=0, qkv=at, cos=0, sin=0, t=0, size=p._APPEND.size):
        return lib.cv3_paged_append(p._APPEND.pack(size, qkv, t, rows, ldq, cos, sin, 0, 0, 0, 4, 2, dim, at, at, at, 0, 2048,
                                                   1024, 64, 2048, 1024, 64, 9, 16, 0), None)
    assert append() == 0
    assert append(dim=72) == U and append(ldq=500) == V and append(ldq=8 * 64 + 2) == V and append(t=3) == V
    assert append(qkv=at + 8) == V and append(cos=at) == V and append(size=0) == V

    def extend(tokens=4, ps=16, cols=3, ld=3, cap=9, size=p._EXTEND.size):
        return lib.cv3_paged_extend(p._EXTEND.pack(size, 0, 0, 0, 2, 0, ld, cols, ps, 0, cap, 0, tokens, *[0] * 7), None)
    assert extend(ps=0) == V and extend(tokens=-1) == V and extend(ld=2) == V and extend(tokens=1 << 31) == V
    assert extend(cols=1 << 28, ld=1 << 28) == V and extend(cap=-1) == V and extend(size=152) == V

    def beam(beams=4, vocab=100, ld=100, stop=(0, 0), t=0, groups=2, ws=0, words=0, size=p._BEAM.size):
        return lib.cv3_beam_select(p._BEAM.pack(size, 0, t, ld, groups, beams, vocab, 0, 0, 0, *stop, *[0] * 6, ws, words, 0.0),
                                   None)
    assert beam(groups=0) == 0
    assert beam(beams=33) == U and beam(beams=0) == U and beam(ld=99) == V and beam(stop=(5, 4)) == V and beam(t=9) == V
    assert beam(groups=40000) == U and beam(size=1) == V
    need = lib.cv3_beam_workspace(1, 32, 10 ** 7)
    assert need > 0 and beam(groups=1, beams=32, vocab=10 ** 7, ld=10 ** 7, ws=at, words=need - 1) == V
    assert b"workspace" in lib.cv3_last_error()
    assert beam(groups=1, beams=32, vocab=10 ** 7, ld=10 ** 7, ws=at + 4, words=need) == V

    def reorder(beams=4, dim=64, st=64, t=0, groups=0, size=p._REORDER.size):
        s = (1 << 16, 2048, 1024, st)
        return lib.cv3_paged_reorder(p._REORDER.pack(size, at, at, t, 2, 9, 2, 16, dim, *s, *s, 0, 3, 3, 0, 0, groups, beams), None)
    assert reorder() == 0 and reorder(beams=1, groups=3) == 0
    assert reorder(beams=33) == U and reorder(st=63) == V and reorder(dim=62, st=64) == V and reorder(t=4) == V
    assert reorder(size=3) == V
    with pytest.raises(RuntimeError):
        L.check(reorder(beams=33), "cv3_paged_reorder")


def test_more_pairs_than_a_grid_holds():
    L, p = pkg("_lib"), pkg("paged")
    lib, at, H = L.load(), 1 << 20, 1 << 16
    for batch in (1 << 15, 1 << 24):
        block = p._ATTENTION.pack(p._ATTENTION.size, at, 0, 32, 32, at, at, 0, 512, 512, 32, 512, 512, 32, 9, 16, at, 1, 1, at,
                                  batch, H, H, 32, 0, at, 32, 32, 0, 0, at, 1 << 60, 0.1)
        assert lib.cv3_paged_attention(block, None) == L.CV3_ERR_VALUE
        assert b"too many" in lib.cv3_last_error()


@pytest.mark.parametrize("alpha", [float("nan"), float("inf"), -float("inf"), 16.5, -17.0])
def test_length_penalties_whose_powers_leave_64_bits(alpha):
    L, p = pkg("_lib"), pkg("paged")
    lib = L.load()
    block = p._BEAM.pack(p._BEAM.size, 0, 0, 100, 0, 4, 100, *[0] * 13, alpha)
    assert lib.cv3_beam_select(block, None) == L.CV3_ERR_VALUE and b"length penalty" in lib.cv3_last_error()
    for fine in (0.0, -16.0, 16.0):
        assert lib.cv3_beam_select(p._BEAM.pack(p._BEAM.size, 0, 0, 100, 0, 4, 100, *[0] * 13, fine), None) == 0


def test_one_hypothesis_of_several_is_evenly_spaced(ops):
    import torch
    one = dict(logits=torch.zeros(3, 5, 50)[:, 2:3], scores=torch.zeros(3, 1), counts=_i32(3, 1), done=_i32(3, 1))
    with pytest.raises(AssertionError, match="accepted"):
        ops.beam_select(**one)


def test_oracle_extend_and_reorder_by_hand():
    """The restatement itself on cases small enough to write down."""
    t = np.array([[4, -1], [5, 6]], np.int32)
    s = np.array([0, 1, 2, 3, 9, 9], np.int32)
    tables, stack, slots, seq, pos, off, lens, count = ref.extend([2, 3], [3, 1], t, s, 4, 2, 5, [0, 1])
    assert tables.tolist() == [[4, 6], [5, 6]] or tables.tolist() == [[4, -1], [5, 6]]
    # request 0 needs two more pages than its two columns hold: nobody is served
    assert lens.tolist() == [2, 0] and off.tolist() == [0, 0, 0] and count == 6 and stack.tolist() == [0, 1, 2, 3, 5, 6]
    tables, stack, slots, seq, pos, off, lens, count = ref.extend([2, 3], [2, 1], t, s, 4, 2, 5, [0, 1])
    assert tables.tolist() == [[4, 6], [5, 6]] and lens.tolist() == [4, 1] and count == 4
    assert slots.tolist() == [12, 13, 10, -1, -1] and seq.tolist() == [0, 0, 1, -1, -1] and pos.tolist() == [2, 3, 0, 0, 0]
    k = np.arange(2 * 3 * 2, dtype=np.float32).reshape(1, 6, 1, 2, 1)
    kk, vv, tt = ref.reorder(k, k, np.array([[0, 1, 2], [3, 4, 5]], np.int32), np.array([[1, 1]], np.int32), [3, 3])
    assert tt.tolist() == [[3, 1, 2], [3, 4, 5]]
    assert kk[0, 1, 0, :, 0].tolist() == [8, 3] and kk[0, 4, 0, :, 0].tolist() == [8, 9]


def test_oracle_beam_against_torch():
    import torch
    rng = np.random.default_rng(0)
    x = rng.normal(size=(2, 3, 40))
    s = rng.normal(size=(2, 3)).astype(np.float32)
    z = np.zeros((2, 3), np.int32)
    tok, par, sc, cnt, done = ref.beam(x, s, z, z, (35, 40))
    cum = torch.log_softmax(torch.from_numpy(x), -1) + torch.from_numpy(s)[..., None].double()
    v, i = cum.view(2, -1).topk(3)
    assert np.array_equal(par * 40 + tok, i.numpy()) and np.allclose(sc, v.numpy(), rtol=1e-12)
    assert np.all(cnt == 1) and np.array_equal(done, tok >= 35)


def test_oracle_attention_against_torch():
    import torch
    rng = np.random.default_rng(0)
    k, v = rng.normal(size=(2, 5, 2, 4, 8))
    t = np.array([[3, 1, 0], [4, 2, 9]], np.int32)
    q = rng.normal(size=(2, 4, 8))
    out, lse = ref.attention(q, k, v, t, [11, 8], 0.3, 6)
    for b, (lo, n) in enumerate(((5, 11), (2, 8))):
        for h in range(4):
            kk = torch.from_numpy(np.concatenate([k[p, h // 2] for p in t[b, :-(-n // 4)]])[lo:n])
            vv = torch.from_numpy(np.concatenate([v[p, h // 2] for p in t[b, :-(-n // 4)]])[lo:n])
            a = 0.3 * (kk @ torch.from_numpy(q[b, h]))
            assert np.allclose(out[b, h], (torch.softmax(a, 0) @ vv).numpy())
            assert np.isclose(lse[b, h], float(torch.logsumexp(a, 0)))


@pytest.mark.parametrize("cos,sin,code", [(0, 0, 0), (0, 16, 0), (4, 0, 1), (0, 8, 1), (12, 12, 1)])
def test_rotation_tables_off_16_byte_boundaries(cos, sin, code):
    """The tables are read 16 bytes at a time: a contiguous view that begins elsewhere is refused."""
    L, p = pkg("_lib"), pkg("paged")
    lib, at = L.load(), 1 << 20
    rc = lib.cv3_paged_append(p._APPEND.pack(p._APPEND.size, at, 0, 0, 512, at + cos, at + sin, 50, at, at, 4, 2, 64, at, at, at,
                                             0, 2048, 1024, 64, 2048, 1024, 64, 9, 16, 0), None)
    assert rc == (L.CV3_ERR_VALUE if code else 0)
    assert not code or b"16-byte" in lib.cv3_last_error()


@pytest.mark.parametrize("pages,ps,code", [(9, (1 << 31) - 1, 0), (9, 1 << 31, 1), (9, 1 << 32, 1), (1 << 31, 16, 1),
                                           ((1 << 31) - 1, 16, 0)])
def test_pages_and_rows_of_a_page_are_32_bit_numbers(pages, ps, code):
    """A slot is divided by the page size in 32 bits where the slot fits in them."""
    L, p = pkg("_lib"), pkg("paged")
    lib, at = L.load(), 1 << 20
    rc = lib.cv3_paged_append(p._APPEND.pack(p._APPEND.size, at, 0, 0, 512, 0, 0, 0, at, 0, 4, 2, 64, at, at, at, 0, 2048, 1024, 64,
                                             2048, 1024, 64, pages, ps, 0), None)
    assert rc == (L.CV3_ERR_VALUE if code else 0)
    assert not code or b"32-bit" in lib.cv3_last_error()


# ---------------------------------------------------------------------------
# pages that several rows name
# ---------------------------------------------------------------------------

def test_oracle_gives_shared_pages_back_once():
    """Two beams of two full pages each both follow the first and are released together: the pages that the second left
    go back when it follows, the shared ones one time when both are released, in the order of their places."""
    t = np.array([[0, 1], [2, 3]], np.int32)
    none, par = np.full(4, -1, np.int32), np.array([[0, 0]], np.int32)
    stack, count, shares, lens = ref.give_back(t, np.array([8, 8]), 4, none, 0, np.zeros(4, np.int32), parents=par)
    assert stack[:count].tolist() == [2, 3] and shares.tolist() == [1, 1, 0, 0] and lens.tolist() == [8, 8]
    t[1] = t[0]
    one, n, left, held = ref.give_back(t, lens, 4, stack, count, shares, release=[1, 0])
    assert n == 2 and left.tolist() == [0] * 4 and held.tolist() == [0, 8]
    stack, count, shares, lens = ref.give_back(t, lens, 4, stack, count, shares, release=[1, 1])
    assert stack[:count].tolist() == [2, 3, 0, 1] and shares.tolist() == [0] * 4
    tables, stack, slots, *_ = ref.extend(lens, [8, 8], t, stack, count, 4, 16)
    assert sorted(tables.reshape(-1).tolist()) == [0, 1, 2, 3] and len(set(slots.tolist())) == 16


def test_refusals_of_shared_pages(ops):
    import torch
    good = dict(lens=_i32(3), new_lens=_i32(3), block_tables=_i32(3, 5), free_pages=_i32(9), free_count=_i32(1),
                page_size=16, max_tokens=4, release=_i32(3), shares=_i32(9))
    with pytest.raises(AssertionError, match="accepted"):
        ops.paged_extend(**good)
    for bad in (torch.zeros(9), torch.zeros(9, dtype=torch.int64), _i32(18)[::2]):
        with pytest.raises(ValueError, match="shares"):
            ops.paged_extend(**{**good, "shares": bad})
    pool = torch.zeros(2, 9, 2, 16, 64)
    fine = dict(k_pages=pool, v_pages=pool, block_tables=_i32(6, 3), parents=_i32(2, 3), lens=_i32(6), shares=_i32(9),
                free_pages=_i32(9), free_count=_i32(1))
    with pytest.raises(AssertionError, match="accepted"):
        ops.paged_reorder(**fine)
    for change in (dict(shares=_i32(8)), dict(shares=torch.zeros(9)), dict(free_pages=torch.zeros(9)), dict(free_count=_i32(2))):
        with pytest.raises(ValueError):
            ops.paged_reorder(**{**fine, **change})
    for gone in ("shares", "free_pages", "free_count"):
        with pytest.raises(ValueError, match="go together"):
            ops.paged_reorder(**{**fine, gone: None})


def test_entry_for_shared_pages():
    """The parameter block has the header's fields, and what is refused is refused before any device work."""
    L, p = pkg("_lib"), pkg("paged")
    lib, at = L.load(), 1 << 20
    text = open(os.path.join(REPO, "include", "cv3cuda.h")).read()
    body = re.search(r"typedef struct cv3_paged_give_back_params \{(.*?)\}", text, re.S).group(1)
    fields = [x.strip() for line in body.split(";") for x in line.split(",") if x.strip()]
    assert p._GIVE_BACK.size == 8 * len(fields) and p._GIVE_BACK.format.lstrip("=") == "%dq" % len(fields)

    def give_back(size=p._GIVE_BACK.size, pages=9, ld=3, cols=3, ps=16, rows=4, release=at, lens_out=at, parents=0, beams=0, cap=9):
        return lib.cv3_paged_give_back(p._GIVE_BACK.pack(size, at, pages, at, ld, cols, ps, at, rows, release, lens_out, parents,
                                                         beams, at, cap, at, at, at), None)
    V, U = L.CV3_ERR_VALUE, L.CV3_ERR_UNSUPPORTED
    assert give_back(size=8) == V and give_back(ld=2) == V and give_back(ps=0) == V and give_back(cap=-1) == V
    assert give_back(release=0) == V and give_back(parents=at) == V and give_back(lens_out=0) == V
    assert give_back(release=0, parents=at, beams=3) == V and give_back(release=0, parents=at, beams=64, rows=64) == U
    assert give_back(release=0, parents=at, beams=2, rows=1 << 18) == U
    assert give_back(rows=1 << 20, cols=1 << 11, ld=1 << 11) == V and give_back(cols=1 << 28, ld=1 << 28) == V
    assert give_back(pages=1 << 31) == V


# ---------------------------------------------------------------------------
# the extension module is a short cut, nothing depends on it
# ---------------------------------------------------------------------------

def _fake_tree(monkeypatch, tmp_path, cxx):
    """A source tree of one kernel file and one binding, compilers that only touch their output (or fail)."""
    b = pkg("build")
    (tmp_path / "csrc" / "bind").mkdir(parents=True)
    (tmp_path / "csrc" / "a.cu").write_text("")
    (tmp_path / "csrc" / "bind" / "x_bind.cpp").write_text("")
    tool = tmp_path / "tool"
    tool.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do if [ "$1" = -o ]; then touch "$2"; fi; shift; done\n')
    broken = tmp_path / "broken"
    broken.write_text("#!/bin/sh\necho 'no headers here' >&2\nexit 1\n")
    for f in (tool, broken):
        f.chmod(0o755)
    for name, value in (("HERE", str(tmp_path)), ("CSRC", str(tmp_path / "csrc")), ("BUILD", str(tmp_path / "_build")),
                        ("LIB", str(tmp_path / "lib.so")), ("NVCC", str(tool))):
        monkeypatch.setattr(b, name, value)
    monkeypatch.setenv("CXX", str(tool if cxx else broken))
    return b


def test_a_binding_that_does_not_compile_leaves_the_library(monkeypatch, tmp_path):
    b = _fake_tree(monkeypatch, tmp_path, False)
    with pytest.warns(UserWarning, match="no headers here"):
        lib = b.build()
    assert os.path.exists(lib) and not [f for f in os.listdir(tmp_path) if "x_bind" in f]


def test_a_binding_belongs_to_one_pytorch(monkeypatch, tmp_path):
    """Its file is named after the PyTorch and the Python that it was built against; another one's is not taken for it."""
    import importlib.metadata
    b = _fake_tree(monkeypatch, tmp_path, True)
    src = str(tmp_path / "csrc" / "bind" / "x_bind.cpp")
    b.build()
    here = b.bind_path(src)
    assert os.path.exists(here) and os.path.basename(here).startswith("_x_bind.") and here.endswith(".so")
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "99.1+other")
    other = b.bind_path(src)
    assert other != here and not os.path.exists(other)
    b.build()
    assert os.path.exists(other) and os.path.exists(here)


def test_a_binding_that_does_not_load_is_left_out(monkeypatch, tmp_path):
    p = pkg("paged")
    file = tmp_path / "_paged_bind.so"
    file.write_bytes(b"not a library")
    monkeypatch.setattr(p, "bind_path", lambda src: str(file), raising=False)
    monkeypatch.setattr(p, "_bound", None)
    with pytest.warns(UserWarning, match="_paged_bind"):
        assert p._bind() is False
    assert p._bind() is False                     # (and says so once)
    with pytest.raises(ValueError, match="CUDA tensors are expected"):
        p.paged_extend(_i32(2), _i32(2), _i32(2, 3), _i32(9), _i32(1), 16, 4)


def test_vocabularies_past_27_bits():
    L, p = pkg("_lib"), pkg("paged")
    lib = L.load()
    for vocab, code in ((1 << 27, 0), ((1 << 27) + 1, L.CV3_ERR_UNSUPPORTED)):
        assert lib.cv3_beam_select(p._BEAM.pack(p._BEAM.size, 0, 0, vocab, 0, 4, vocab, *[0] * 13, 0.0), None) == code
