"""Operators of the paged key/value cache and of beam search (re-exported by :mod:`.ops`).

A cache layer is a pool of pages ``(pages, kv_heads, page_size, head_dim)`` for keys and one for
values; a transposed view of ``(pages, page_size, kv_heads, head_dim)`` serves as well (rows of
``head_dim`` elements stay contiguous).  A request's pages are named by its row of ``block_tables``
(int32), and a *slot* is ``page * page_size + row``.  The operators chain into a decode step::

    step = ops.paged_extend(lens, new_lens, block_tables, free_pages, free_count, page_size, max_tokens)
    q = ops.paged_append(qkv, step.slots, step.pos, k_pages, v_pages, heads, cos, sin)
    out = ops.paged_attention(q, k_pages, v_pages, block_tables, step.lens)
    ...                                                # the other layers, the head
    best = ops.beam_select(logits, scores, counts, done, stop=(6561, 6761))
    ops.paged_reorder(k_all, v_all, block_tables, best.parents, step.lens, shares, free_pages, step.free_count)

Beams share pages; ``shares`` counts them, so that each goes back to the stack once, when no row names
it any more.  Pools, tables and state are updated in place, so every argument is a device array; a host array
raises ValueError.  Shape, type and alignment errors raise ValueError, configurations that are not
built RuntimeError.  The calls are ordered on the current stream of the current device (on which
all arrays have to be), take no persistent workspace and can be captured into a CUDA graph: what
they read on the device (lengths, tables, flags) may change between replays.
"""

from __future__ import annotations

import ctypes
import importlib.util
import math
import os
import struct
import warnings
from typing import NamedTuple, Optional, Tuple

import numpy as np

from . import _dev as D
from ._lib import check, load
from .build import bind_path

torch = D.torch

MAX_BEAMS = 32   # CV3_MAX_BEAMS

# The C entries' parameter blocks (include/cv3cuda.h): 64-bit fields, packed here in one call -- a
# third of what 20 to 35 ctypes arguments cost.
_EXTEND, _APPEND, _ATTENTION, _BEAM, _REORDER, _GIVE_BACK = (struct.Struct("=" + f) for f in
                                                             ("20q", "26q", "32qd", "20qd", "24q", "18q"))

if torch is not None:
    _TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
else:
    _TYPES = {np.dtype(np.float32): 0, np.dtype(np.float16): 1}


class PagedStep(NamedTuple):
    """What :func:`paged_extend` gives: one row per new token, and the new state."""
    slots: object        # int64 (max_tokens,), -1 behind the last token
    seq: object          # int32 (max_tokens,) request of the token, -1 behind the last
    pos: object          # int32 (max_tokens,) its position in the request
    offsets: object      # int32 (batch + 1,) rows of request b: offsets[b] .. offsets[b + 1]
    lens: object         # int32 (batch,) tokens held, the new ones included
    free_count: object   # int32 (1,) pages left on the stack


class BeamStep(NamedTuple):
    """What :func:`beam_select` gives, ``(groups, beams)`` each, best first."""
    tokens: object       # int64
    parents: object      # int32
    scores: object       # float32
    counts: object       # int32
    done: object         # int32


_bound = None   # the short way (csrc/bind/paged_bind.cpp), False where there is none


def _bind():
    """The extension module that takes plain calls of PyTorch tensors; False without PyTorch or without
    a module built against it (every call then goes the long way, which gives the same results)."""
    global _bound
    if _bound is None:
        _bound = False
        path = bind_path("paged_bind.cpp") if torch is not None else ""
        if os.path.exists(path):
            try:
                spec = importlib.util.spec_from_file_location("_paged_bind", path)
                mod = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(mod)
            except (ImportError, OSError, SystemError) as e:
                warnings.warn(f"{path} does not load, the paged operators take the long way: {e}")
                return _bound
            lib = load()
            mod.setup(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in
                        ("cv3_paged_extend", "cv3_paged_append", "cv3_paged_attention", "cv3_paged_attention_workspace",
                         "cv3_beam_select", "cv3_beam_workspace", "cv3_paged_reorder")), PagedStep, BeamStep)
            _bound = mod
    return _bound


def _new(like, shape, dtype):
    """An uninitialised array next to ``like``."""
    return like.new_empty(shape, dtype=dtype) if torch is not None else D.empty(shape, dtype)


def _device(name: str, *arrays) -> int:
    """The device of the arrays: all on the current one, or ValueError."""
    if torch is None:
        for x in arrays:
            if not isinstance(x, D.DeviceArray):
                raise ValueError(f"{name}: device arrays are expected, got {type(x).__name__}")
        D.require_cuda()
        return 0
    here = -2
    for x in arrays:
        try:
            at = x.get_device()
        except AttributeError:
            at = -1
        if at < 0:
            raise ValueError(f"{name}: CUDA tensors are expected, got a host {type(x).__name__}")
        if here == -2:
            here = at
        elif at != here:
            raise ValueError(f"{name}: tensors on cuda:{here} and cuda:{at}")
    if here != torch.cuda.current_device():
        raise ValueError(f"{name}: tensors on cuda:{here}, the current device is cuda:{torch.cuda.current_device()}")
    return here


def _ints(name: str, what: str, x, n: int, dtype=None) -> int:
    """Pointer of ``n`` contiguous int32 (or ``dtype``) values."""
    if x.dtype != (D.I32 if dtype is None else dtype) or x.numel() != n or not x.is_contiguous():
        raise ValueError(f"{name}: {what} must be {n} contiguous {'int32' if dtype is None else dtype} values, got "
                         f"{tuple(x.shape)} {x.dtype}")
    return x.data_ptr()


def _table(name: str, tables, rows: Optional[int]) -> Tuple[int, int, int]:
    """(pointer, row stride, columns) of an int32 block table."""
    shape, st = tables.shape, tables.stride()
    if len(shape) != 2 or tables.dtype != D.I32 or (rows is not None and shape[0] != rows) \
            or (shape[0] > 0 and shape[1] > 1 and st[1] != 1):
        raise ValueError(f"{name}: block_tables must be int32 (requests, blocks) with contiguous rows, got "
                         f"{tuple(shape)} {tables.dtype}")
    return tables.data_ptr(), st[0] if shape[0] > 1 else max(st[0], shape[1]), shape[1]


def _type(name: str, x) -> int:
    t = _TYPES.get(x.dtype)
    if t is None:
        raise ValueError(f"{name}: float32, float16 or bfloat16 expected, got {x.dtype}")
    return t


def _pools(name: str, k, v, dims: int, written: bool = False):
    """(type, shape, k strides, v strides) of a pair of page pools with contiguous rows."""
    shape, ks, vs = k.shape, k.stride(), v.stride()
    if len(shape) != dims or tuple(v.shape) != tuple(shape) or v.dtype != k.dtype:
        raise ValueError(f"{name}: k_pages and v_pages must be alike, {dims}-dimensional "
                         f"(..., kv_heads, page_size, head_dim), got {tuple(shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    if ks[-1] != 1 or vs[-1] != 1:
        raise ValueError(f"{name}: the rows of head_dim elements must be contiguous")
    if min(ks) < 0 or min(vs) < 0 or shape[-2] == 0 or shape[-3] == 0:
        raise ValueError(f"{name}: empty or reversed page dimensions")
    if written and any(n > 1 and (a == 0 or b == 0) for n, a, b in zip(shape, ks, vs)):
        raise ValueError(f"{name}: pools that are written cannot be expanded views")
    return _type(name, k), shape, ks, vs


def _like(name: str, out, shape, dtype):
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or not out.is_contiguous():
        raise ValueError(f"{name}: out must be contiguous {tuple(shape)} {dtype}, got {tuple(out.shape)} {out.dtype}")
    return out


def _give_back(name, d, shares, tables, lens, n, page_size, free_pages, free_count, count_out, release=0, lens_out=0, parents=0,
               beams=0):
    """Rows leave their pages (cv3_paged_give_back); pointers but for the arrays shares, lens and free_pages."""
    tp, ld, cols = tables
    scratch = _new(lens, (n,), D.I32)
    rc = load().cv3_paged_give_back(
        _GIVE_BACK.pack(_GIVE_BACK.size, _ints(name, "shares", shares, shares.numel()), shares.numel(), tp, ld, cols, page_size,
                        lens.data_ptr(), n, release, lens_out, parents, beams, free_pages.data_ptr(), free_pages.numel(),
                        free_count, count_out, scratch.data_ptr()), D.raw_stream(d))
    if rc:
        check(rc, name)


def paged_extend(lens, new_lens, block_tables, free_pages, free_count, page_size: int, max_tokens: int, release=None,
                 out: Optional[PagedStep] = None, shares=None) -> PagedStep:
    """Cache pages and slots for the new tokens of every request.

    Request ``b`` holds ``lens[b]`` tokens (int32) and gets ``new_lens[b]`` more; where ``release[b]``
    is not 0 it first gives its pages back and starts from none, so a finished request's place serves
    the next one in the same call.  ``free_pages[:free_count]`` is the stack of free page numbers
    (updated in place, as is ``block_tables``).  Requests are served in order; from the first whose
    pages, rows (``max_tokens`` over all) or table columns do not suffice on, none gets new tokens.
    Returns a :class:`PagedStep`, whose rows behind the last token have slot -1; ``out`` gives it its tensors (``out.lens`` may be ``lens`` and
    ``out.free_count`` may be ``free_count``: the state then advances in place).

    ``shares`` (int32, one number per page of the pool, zeros to begin with, updated in place) holds for
    every page the rows that name it beyond the first, as :func:`paged_reorder` leaves them: a released
    row then gives back the pages that no other row names.  Without it every page of a released row goes
    back, so rows that share pages must not be released.
    """
    if out is None and shares is None and (_bound or _bind()):
        r = _bound.extend(lens, new_lens, block_tables, free_pages, free_count, page_size, max_tokens, release)
        if r is not None:
            return r
    name = "paged_extend"
    arrays = (lens, new_lens, block_tables, free_pages, free_count)
    d = _device(name, *arrays, *(x for x in (release, shares) if x is not None))
    if len(lens.shape) != 1:
        raise ValueError(f"{name}: lens must be (requests,), got {tuple(lens.shape)}")
    n, T = lens.shape[0], int(max_tokens)
    if page_size <= 0 or not 0 <= T < 2 ** 31 - 1024:
        raise ValueError(f"{name}: page_size {page_size}, max_tokens {max_tokens}")
    pl, pn = _ints(name, "lens", lens, n), _ints(name, "new_lens", new_lens, n)
    pr = 0 if release is None else _ints(name, "release", release, n)
    tp, ld, cols = _table(name, block_tables, n)
    cap = free_pages.numel()
    pf, pc = _ints(name, "free_pages", free_pages, cap), _ints(name, "free_count", free_count, 1)
    if shares is not None:
        _ints(name, "shares", shares, shares.numel())
    if out is None:
        sizes = (T, T, n + 1, n, 1, n + 1)
        if torch is not None:
            parts = torch.split_with_sizes(lens.new_empty((2 * T + 3 * n + 3,)), sizes)
        else:
            parts = [D.empty((m,), D.I32) for m in sizes]
        out = PagedStep(_new(lens, (T,), D.I64), *parts[:5])
        scratch = parts[5]
    else:
        _device(name, lens, *out)
        _ints(name, "out.slots", out.slots, T, D.I64)
        for what, x, m in (("seq", out.seq, T), ("pos", out.pos, T), ("offsets", out.offsets, n + 1),
                           ("lens", out.lens, n), ("free_count", out.free_count, 1)):
            _ints(name, "out." + what, x, m)
        scratch = _new(lens, (n + 1,), D.I32)
    if shares is not None and release is not None and n:
        held, left = _new(lens, (n,), D.I32), _new(lens, (1,), D.I32)
        _give_back(name, d, shares, (tp, ld, cols), lens, n, page_size, free_pages, pc, left.data_ptr(), release=pr,
                   lens_out=held.data_ptr())
        pl, pr, pc = held.data_ptr(), 0, left.data_ptr()
    rc = load().cv3_paged_extend(
        _EXTEND.pack(_EXTEND.size, pl, pn, pr, n, tp, ld, cols, page_size, pf, cap, pc, T, out.slots.data_ptr(),
                     out.seq.data_ptr(), out.pos.data_ptr(), out.offsets.data_ptr(), out.lens.data_ptr(),
                     out.free_count.data_ptr(), scratch.data_ptr()), D.raw_stream(d))
    if rc:
        check(rc, name)
    return out


def paged_append(qkv, slots, pos, k_pages, v_pages, heads: int, cos=None, sin=None, out=None, bad=None):
    """RoPE of fused qkv rows and the store of their keys and values by slot.

    ``qkv`` ``(rows, (heads + 2 * kv_heads) * head_dim)`` holds query, key and value heads; returns the
    rotated queries ``(rows, heads, head_dim)`` in its type and writes keys (rotated) and values in the
    pools' type at ``slots`` (int64; -1: not stored).  ``cos`` / ``sin`` are fp32 ``(positions,
    head_dim)`` half-split tables on 16-byte boundaries, read at ``pos`` (int32); without them nothing is
    rotated and ``pos`` may be None.  A slot outside the pool, or a position outside the tables, stores nothing and counts
    into ``bad`` (int32, one value).  The slots of one call must differ.
    """
    if _bound or _bind():
        r = _bound.append(qkv, slots, pos, k_pages, v_pages, heads, cos, sin, out, bad)
        if r is not None:
            return r
    name = "paged_append"
    d = _device(name, qkv, slots, k_pages, v_pages, *(x for x in (pos, cos, sin, out, bad) if x is not None))
    kt, shape, ks, vs = _pools(name, k_pages, v_pages, 4, True)
    pages, kv, ps, dim = shape
    t = _type(name, qkv)
    if qkv.dim() != 2 or heads <= 0 or qkv.shape[1] != (heads + 2 * kv) * dim:
        raise ValueError(f"{name}: qkv rows of ({heads} + 2 * {kv}) * {dim} elements expected, got {tuple(qkv.shape)}")
    rows, (ldq, one) = qkv.shape[0], qkv.stride()
    if one != 1:
        raise ValueError(f"{name}: qkv rows must be contiguous")
    pslots = _ints(name, "slots", slots, rows, D.I64)
    pc = psn = positions = 0
    if (cos is None) != (sin is None) or (cos is not None and pos is None):
        raise ValueError(f"{name}: cos, sin and pos go together")
    ppos = 0 if pos is None else _ints(name, "pos", pos, rows)
    if cos is not None:
        positions = cos.shape[0]
        for x in (cos, sin):
            if x.dtype != D.F32 or tuple(x.shape) != (positions, dim) or not x.is_contiguous():
                raise ValueError(f"{name}: cos and sin must be contiguous float32 (positions, {dim})")
        pc, psn = cos.data_ptr(), sin.data_ptr()
    if out is None:
        out = _new(qkv, (rows, heads, dim), qkv.dtype)
    else:
        _like(name, out, (rows, heads, dim), qkv.dtype)
    pbad = 0 if bad is None else _ints(name, "bad", bad, 1)
    rc = load().cv3_paged_append(
        _APPEND.pack(_APPEND.size, qkv.data_ptr(), t, rows, ldq if rows > 1 else qkv.shape[1], pc, psn, positions, pslots,
                     ppos, heads, kv, dim, out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), kt, ks[0], ks[1],
                     ks[2], vs[0], vs[1], vs[2], pages, ps, pbad), D.raw_stream(d))
    if rc:
        check(rc, name)
    return out


def paged_attention(q, k_pages, v_pages, block_tables, lens, scale: Optional[float] = None, window: int = 0, out=None,
                    return_lse: bool = False, bad=None):
    """Softmax attention of one new token per request over its cached tokens.

    ``q`` ``(batch, heads, head_dim)`` -> the same shape and type; GQA when the pools have fewer heads;
    the pools may have another element type (an fp16 or bf16 cache under fp32 activations keeps fp32
    arithmetic).  ``lens`` (int32) counts the cached tokens, the new one included; ``window`` > 0 keeps
    the last ``window`` of them.  A request without tokens gives zeros.  ``return_lse`` adds the fp32
    ``(batch, heads)`` logarithms of the softmax sums (-inf without tokens), by which results over
    separate caches are joined.  Tokens of a page number outside the pool are left out and counted
    (per table entry) into ``bad``.
    """
    if _bound or _bind():
        r = _bound.attention(q, k_pages, v_pages, block_tables, lens, scale, window, out, return_lse, bad)
        if r is not None:
            return r
    name = "paged_attention"
    d = _device(name, q, k_pages, v_pages, block_tables, lens, *(x for x in (out, bad) if x is not None))
    kt, shape, ks, vs = _pools(name, k_pages, v_pages, 4)
    pages, kv, ps, dim = shape
    qt = _type(name, q)
    if q.dim() != 3 or q.shape[2] != dim:
        raise ValueError(f"{name}: q must be (batch, heads, {dim}), got {tuple(q.shape)}")
    B, H = q.shape[0], q.shape[1]
    if H == 0 or H % kv:
        raise ValueError(f"{H} query heads is not a multiple of {kv} kv heads")
    qsb, qsh, one = q.stride()
    if one != 1:
        raise ValueError(f"{name}: the heads of q must be contiguous")
    window = int(window)
    if window < 0:
        raise ValueError(f"{name}: window {window}")
    tp, ld, cols = _table(name, block_tables, B)
    plens = _ints(name, "lens", lens, B)
    if out is None:
        out = _new(q, (B, H, dim), q.dtype)
    else:
        _like(name, out, (B, H, dim), q.dtype)
    pbad = 0 if bad is None else _ints(name, "bad", bad, 1)
    lse = _new(q, (B, H), D.F32) if return_lse else None
    lib = load()
    words = lib.cv3_paged_attention_workspace(B, H, kv, dim, kt, cols * ps)
    ws = _new(q, (words,), D.F32) if words else None
    rc = lib.cv3_paged_attention(
        _ATTENTION.pack(_ATTENTION.size, q.data_ptr(), qt, qsb, qsh, k_pages.data_ptr(), v_pages.data_ptr(), kt, ks[0],
                        ks[1], ks[2], vs[0], vs[1], vs[2], pages, ps, tp, ld, cols, plens, B, H, kv, dim, window,
                        out.data_ptr(), H * dim, dim, lse.data_ptr() if return_lse else 0, pbad,
                        ws.data_ptr() if words else 0, words, 1.0 / math.sqrt(dim) if scale is None else scale),
        D.raw_stream(d))
    if rc:
        check(rc, name)
    return (out, lse) if return_lse else out


def beam_select(logits, scores, counts, done, stop: Optional[Tuple[int, int]] = None, min_len=None,
                length_penalty: float = 0.0, out: Optional[BeamStep] = None) -> BeamStep:
    """The best continuations of every group's hypotheses.

    ``logits`` ``(groups, beams, vocab)``; ``scores`` (float32 sums of log-probabilities), ``counts``
    and ``done`` (int32) are ``(groups, beams)``.  A candidate's key is its new score divided by its
    length to the power ``length_penalty`` (-16 to 16); the ``beams`` best of all ``beams * vocab`` are kept, equal
    keys go to the lower hypothesis, its larger logit, the lower token.  A token in ``stop`` (first, end) finishes a
    hypothesis, and is no candidate while it has fewer than ``min_len[group]`` tokens; a finished one
    stays as it is (token 0).  A score of -inf marks a hypothesis that does not exist, as all but the
    first at the start.  NaN logits are no candidates.  Keys are computed in 64 bits, from
    log-sum-exps held to 2e-8.
    ``out`` gives the :class:`BeamStep` its tensors, which may be the input state.
    """
    if out is None and (_bound or _bind()):
        r = _bound.beam(logits, scores, counts, done, stop, min_len, length_penalty)
        if r is not None:
            return r
    name = "beam_select"
    d = _device(name, logits, scores, counts, done, *((min_len,) if min_len is not None else ()))
    t = _type(name, logits)
    if logits.dim() != 3:
        raise ValueError(f"{name}: logits must be (groups, beams, vocab), got {tuple(logits.shape)}")
    G, K, V = logits.shape
    sg, sk, sv = logits.stride()
    if K == 1:
        sk = sg
    if (V > 1 and sv != 1) or (G > 1 and sg != K * sk):
        raise ValueError(f"{name}: rows of logits must be contiguous and evenly spaced")
    n = G * K
    for what, x, dt in (("scores", scores, D.F32), ("counts", counts, D.I32), ("done", done, D.I32)):
        if x.dtype != dt or x.shape != (G, K) or not x.is_contiguous():
            raise ValueError(f"{name}: {what} must be contiguous ({G}, {K}) {dt}, got {tuple(x.shape)} {x.dtype}")
    pc, pd = counts.data_ptr(), done.data_ptr()
    pm = 0 if min_len is None else _ints(name, "min_len", min_len, G)
    lo, hi = (0, 0) if stop is None else stop
    if not 0 <= lo <= hi <= V:
        raise ValueError(f"{name}: stop tokens {lo}..{hi} outside the vocabulary of {V}")
    if out is None:
        out = BeamStep(_new(counts, (G, K), D.I64), D.empty_like(counts), D.empty_like(scores), D.empty_like(counts),
                       D.empty_like(done))
    else:
        _device(name, logits, *out)
        for x, dt in zip(out, (D.I64, D.I32, D.F32, D.I32, D.I32)):
            _like(name, x, (G, K), dt)
    lib = load()
    size = lib.cv3_beam_workspace(G, K, V)
    ws = _new(counts, (size >> 3,), D.I64) if size else None
    rc = lib.cv3_beam_select(
        _BEAM.pack(_BEAM.size, logits.data_ptr(), t, sk if n > 1 else V, G, K, V, scores.data_ptr(), pc, pd, lo, hi, pm,
                   out.tokens.data_ptr(), out.parents.data_ptr(), out.scores.data_ptr(), out.counts.data_ptr(),
                   out.done.data_ptr(), ws.data_ptr() if size else 0, size, length_penalty), D.raw_stream(d))
    if rc:
        check(rc, name)
    return out


def paged_reorder(k_pages, v_pages, block_tables, parents, lens, shares=None, free_pages=None, free_count=None) -> None:
    """The cache follows the beams, in place.

    Pools ``(layers, pages, kv_heads, page_size, head_dim)`` (or one layer without the first
    dimension); ``block_tables`` ``(groups * beams, blocks)``; ``parents`` int32 ``(groups, beams)``;
    ``lens`` int32 ``(groups * beams,)``, alike within a group.  Beam k becomes what beam
    ``parents[g][k]`` was: full pages are shared through the table, the tokens of the last, partly
    filled page are copied into the page that beam k's own row names there (and no other beam's).

    ``shares`` (int32, one number per page: the rows that name it beyond the first), ``free_pages`` and
    ``free_count`` (all three or none, updated in place) keep account of the shared pages: those that no
    beam names any more go back to the stack, and :func:`paged_extend` with ``shares`` may release beams.
    Without them a page that is left stays out of the stack, and beams must not be released.
    """
    counted = tuple(x for x in (shares, free_pages, free_count) if x is not None)
    if not counted and (_bound or _bind()) and _bound.reorder(k_pages, v_pages, block_tables, parents, lens):
        return
    name = "paged_reorder"
    if len(counted) not in (0, 3):
        raise ValueError(f"{name}: shares, free_pages and free_count go together")
    d = _device(name, k_pages, v_pages, block_tables, parents, lens, *counted)
    dims = len(k_pages.shape)
    if dims not in (4, 5):
        raise ValueError(f"{name}: pools of 4 or 5 dimensions expected, got {tuple(k_pages.shape)}")
    kt, shape, ks, vs = _pools(name, k_pages, v_pages, dims, True)
    if dims == 4:
        shape, ks, vs = (1,) + tuple(shape), (0,) + tuple(ks), (0,) + tuple(vs)
    layers, pages, kv, ps, dim = shape
    if len(parents.shape) != 2:
        raise ValueError(f"{name}: parents must be (groups, beams), got {tuple(parents.shape)}")
    G, K = parents.shape
    pp = _ints(name, "parents", parents, G * K)
    tp, ld, cols = _table(name, block_tables, G * K)
    plens = _ints(name, "lens", lens, G * K)
    if counted:
        _ints(name, "shares", shares, pages), _ints(name, "free_pages", free_pages, free_pages.numel())
        pc = _ints(name, "free_count", free_count, 1)
    lib = load()
    block = _REORDER.pack(_REORDER.size, k_pages.data_ptr(), v_pages.data_ptr(), kt, layers, pages, kv, ps, dim, *ks[:4], *vs[:4], tp,
                          ld, cols, pp, plens, G, K)
    if counted:
        # (no groups: what the copy refuses is refused before anything is counted)
        rc = lib.cv3_paged_reorder(block[:-16] + struct.pack("=2q", 0, K), D.raw_stream(d))
        if rc:
            check(rc, name)
        if G > 0 and K > 1:
            _give_back(name, d, shares, (tp, ld, cols), lens, G * K, ps, free_pages, pc, pc, parents=pp, beams=K)
    rc = lib.cv3_paged_reorder(block, D.raw_stream(d))
    if rc:
        check(rc, name)
