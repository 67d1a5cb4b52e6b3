"""The paged key/value cache of the speech LM and beam search over it (no counterpart in the
reference, which keeps one array per sequence and one hypothesis).

:class:`PagedKVCache` holds every layer's pages, the block tables, the stack of free pages and the
requests' lengths on the device; :class:`BeamEngine` advances ``groups * beams`` hypotheses one token
per step, a step -- pages and slots, every layer, the head, the choice, the cache following it and
the next embedding -- being one CUDA graph replay, as in :class:`.qwen2.DecodeEngine`.
"""

from __future__ import annotations

from typing import List, Sequence, Tuple

import numpy as np

from .. import _dev as D
from .. import paged as ops
from .._lib import call
from ..quant import QTensor
from ._common import TC_MIN_ROWS, DecodeGemv, Graph, Lin
from .qwen2 import DecodeEngine, Qwen2Model, decode_gemvs

torch = D.torch


class PagedKVCache:
    """Pages ``(layers, pages, kv_heads, page_size, head_dim)`` of keys and of values for ``requests``
    requests of up to ``max_len`` tokens; ``dtype`` float32, float16 or bfloat16.

    Beams share pages, which ``shares`` counts: a page returns to the stack when no request names it any
    more.  ``releases=False`` saves the counting for a cache whose requests are never released: pages that
    beams leave then stay out of the stack until :meth:`start_beams` begins anew."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, requests: int, max_len: int, pages: int,
                 page_size: int = 16, dtype=None, releases: bool = True):
        dtype = D.F32 if dtype is None else dtype
        self.layers, self.kv_heads, self.head_dim, self.page_size, self.pages = layers, kv_heads, head_dim, page_size, pages
        self.blocks = -(-max_len // page_size)
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.k, self.v = D.zeros(shape, dtype), D.zeros(shape, dtype)
        self.tables = torch.full((requests, self.blocks), -1, dtype=torch.int32, device="cuda")
        self.free = torch.arange(pages, dtype=torch.int32, device="cuda")
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.bad = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.shares = torch.zeros(pages, dtype=torch.int32, device="cuda") if releases else None

    def nbytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()

    def extend(self, new_lens, max_tokens: int, release=None) -> ops.PagedStep:
        """Pages and slots for every request's new tokens (:func:`ops.paged_extend`); the state advances."""
        n, T = self.lens.shape[0], int(max_tokens)
        i32 = dict(dtype=torch.int32, device="cuda")
        out = ops.PagedStep(torch.empty(T, dtype=torch.int64, device="cuda"), torch.empty(T, **i32), torch.empty(T, **i32),
                            torch.empty(n + 1, **i32), self.lens, self.free_count)
        return self.extend_into(out, new_lens, release)

    def extend_into(self, out: ops.PagedStep, new_lens, release=None) -> ops.PagedStep:
        if release is not None and self.shares is None:
            raise ValueError("a cache made with releases=False releases no requests")
        return ops.paged_extend(self.lens, new_lens, self.tables, self.free, self.free_count, self.page_size,
                                out.slots.shape[0], release=release, out=out, shares=self.shares)

    def append(self, layer: int, qkv, step: ops.PagedStep, heads: int, cos, sin, out=None):
        """Rotated queries of fused rows; their keys and values go to the step's slots."""
        return ops.paged_append(qkv, step.slots, step.pos, self.k[layer], self.v[layer], heads, cos, sin, out=out,
                                bad=self.bad)

    def attention(self, layer: int, q, scale: float, out=None):
        return ops.paged_attention(q, self.k[layer], self.v[layer], self.tables, self.lens, scale=scale, out=out,
                                   bad=self.bad)

    def reorder(self, parents) -> None:
        counts = () if self.shares is None else (self.shares, self.free, self.free_count)
        ops.paged_reorder(self.k, self.v, self.tables, parents, self.lens, *counts)

    def start_beams(self, prompts, cache, beams: int) -> None:
        """Begins ``beams`` hypotheses of every prompt (lengths ``prompts``) from the contiguous prefill
        ``cache``: full pages are shared by a group's rows, each row has a last page of its own."""
        ps, at = self.page_size, 0
        tables, shares = np.full(tuple(self.tables.shape), -1, np.int32), np.zeros(self.pages, np.int32)
        src, dst = [], []      # (group, block) -> page
        for g, n in enumerate(prompts):
            rows = slice(g * beams, (g + 1) * beams)
            full, rest = divmod(n, ps)
            if -(-n // ps) > self.blocks:
                raise ValueError(f"a prompt of {n} tokens in a cache of {self.blocks} pages per request")
            tables[rows, :full] = np.arange(at, at + full)
            shares[at:at + full] = beams - 1
            src += [(g, j) for j in range(full)]
            dst += list(range(at, at + full))
            at += full
            if rest:
                tables[rows, full] = np.arange(at, at + beams)
                src += [(g, full)] * beams
                dst += list(range(at, at + beams))
                at += beams
        if at > self.pages:
            raise ValueError(f"{at} pages for the prompts, {self.pages} in the cache")
        self.tables.copy_(torch.from_numpy(tables))
        if self.shares is not None:
            self.shares.copy_(torch.from_numpy(shares))
        self.free.copy_(torch.arange(self.pages, dtype=torch.int32))
        self.free[:self.pages - at] = torch.arange(self.pages - 1, at - 1, -1, dtype=torch.int32)
        self.free_count.fill_(self.pages - at)
        self.lens.copy_(torch.tensor(list(prompts), dtype=torch.int32).repeat_interleave(beams))
        g, j = (torch.tensor(x, device="cuda") for x in zip(*src))
        to = torch.tensor(dst, device="cuda")
        for mine, theirs in ((self.k, cache.k), (self.v, cache.v)):
            L, B, H, cap, hd = theirs.shape
            blocks = theirs.view(L, B, H, cap // ps, ps, hd)[:, g, :, j]      # (rows, layers, heads, page, dim)
            mine[:, to] = blocks.transpose(0, 1).to(mine.dtype)


class BeamEngine:
    """Beam search of ``groups`` prompts with ``beams`` hypotheses each (``groups * beams`` <= 32: the
    decode GEMV's rows), up to ``max_steps`` tokens after prompts of up to ``max_prompt``."""

    POLL = 8   # steps between two looks at the done flags

    def __init__(self, model: Qwen2Model, head_w, head_bias, speech_emb, stop: Tuple[int, int], groups: int, beams: int,
                 max_prompt: int, max_steps: int, page_size: int = 16, cache_dtype=None, length_penalty: float = 0.0):
        c = model.cfg
        R = groups * beams
        if not 1 <= beams <= ops.MAX_BEAMS:
            raise ValueError(f"{beams} beams: 1 to {ops.MAX_BEAMS} are supported")
        self.m, self.c, self.G, self.K, self.R = model, c, groups, beams, R
        self.stop, self.alpha = stop, float(length_penalty)
        H, Hk, hd, hid = c.num_attention_heads, c.num_key_value_heads, c.head_dim, c.hidden_size
        self.max_prompt, self.max_steps = max_prompt, max_steps
        need = -(-max_prompt // page_size) + beams * (-(-max_steps // page_size) + 2)
        self.cache = PagedKVCache(c.num_hidden_layers, Hk, hd, R, max_prompt + max_steps, groups * need, page_size, cache_dtype,
                                  releases=False)   # (every run begins anew)
        self.head = Lin(head_w, head_bias)
        self.vocab = self.head.n
        self.emb = speech_emb
        self.h = D.zeros((R, hid))
        self.n = D.zeros((R, hid))
        self.qkv = D.zeros((R, (H + 2 * Hk) * hd))
        self.q, self.a = D.zeros((R, H, hd)), D.zeros((R, H, hd))
        self.gu = D.empty((R, 2 * c.intermediate_size))
        self.act = D.empty((R, c.intermediate_size))
        self.logits = D.zeros((groups, beams, self.vocab))
        i32 = dict(dtype=torch.int32, device="cuda")
        self.state = ops.BeamStep(torch.zeros((groups, beams), dtype=torch.int64, device="cuda"),
                                  torch.zeros((groups, beams), **i32), D.zeros((groups, beams)),
                                  torch.zeros((groups, beams), **i32), torch.zeros((groups, beams), **i32))
        self.min_len = torch.zeros(groups, **i32)
        self.ones = torch.ones(R, **i32)
        self.step_out = ops.PagedStep(torch.zeros(R, dtype=torch.int64, device="cuda"), torch.zeros(R, **i32),
                                      torch.zeros(R, **i32), torch.zeros(R + 1, **i32), self.cache.lens,
                                      self.cache.free_count)
        self.tokens = torch.zeros((max_steps, groups, beams), dtype=torch.int64, device="cuda")
        self.parents = torch.zeros((max_steps, groups, beams), **i32)
        self.cos, self.sin = model.rope(max_prompt + max_steps)
        self.scale = float(np.float32(1.0 / np.sqrt(hd)))
        self.fast = decode_gemvs(model, DecodeEngine.QKV_SPLITS)
        self.fast_head = DecodeGemv(head_w, bias=head_bias, norm_w=model.norm_w(), eps=c.rms_norm_eps) \
            if isinstance(head_w, QTensor) and head_w.kind == "q8" else None
        if R >= TC_MIN_ROWS:   # the weight remainders of the tensor-core linears, before any capture
            for lin in [self.head] + [x for L, F in zip(model.layers(), self.fast) if F is None
                                      for x in (L.qkv, L.o, L.gu, L.down)]:
                if not lin.q8:
                    lin.lo()
        self.graph = None

    # -- one step -----------------------------------------------------------------
    def launches(self, st) -> None:
        c, R = self.c, self.R
        hid, H = c.hidden_size, c.num_attention_heads
        h, n, a, act, gu = (t.data_ptr() for t in (self.h, self.n, self.a, self.act, self.gu))
        step = self.cache.extend_into(self.step_out, self.ones)
        for i, L in enumerate(self.m.layers()):
            F = self.fast[i]
            if F is not None:
                F[0](h, R, self.qkv.data_ptr(), stream=st)
            else:
                call("cv3_rms_norm", h, L.ln1.data_ptr(), R, hid, c.rms_norm_eps, n, st)
                L.qkv(n, R, self.qkv.data_ptr(), stream=st)
            self.cache.append(i, self.qkv, step, H, self.cos, self.sin, out=self.q)
            self.cache.attention(i, self.q, self.scale, out=self.a)
            if F is not None:
                F[1](a, R, h, residual=h, stream=st)
                F[2](h, R, act, stream=st)
                F[3](act, R, h, residual=h, stream=st)
            else:
                L.o(a, R, h, residual=h, stream=st)
                call("cv3_rms_norm", h, L.ln2.data_ptr(), R, hid, c.rms_norm_eps, n, st)
                L.gu(n, R, gu, stream=st)
                call("cv3_swiglu", gu, R, c.intermediate_size, act, st)
                L.down(act, R, h, residual=h, stream=st)
        if self.fast_head is not None:
            self.fast_head(h, R, self.logits.data_ptr(), stream=st)
        else:
            call("cv3_rms_norm", h, self.m.norm_w().data_ptr(), R, hid, c.rms_norm_eps, n, st)
            self.head(n, R, self.logits.data_ptr(), stream=st)
        self.choose(st)

    def choose(self, st) -> None:
        """The best continuations, the cache that follows them and the next step's input rows."""
        s = self.state
        ops.beam_select(self.logits, s.scores, s.counts, s.done, stop=self.stop, min_len=self.min_len,
                        length_penalty=self.alpha, out=s)
        self.cache.reorder(s.parents)
        e = self.emb
        quant = isinstance(e, QTensor)
        dim = int(e.shape[1])
        call("cv3_embedding", (e.q if quant else e).data_ptr(), (3 if e.kind == "q4" else 2) if quant else 0,
             e.scales.data_ptr() if quant else None, int(e.shape[0]), dim, e.padded_k if quant else dim,
             s.tokens.data_ptr(), self.R, self.h.data_ptr(), dim, None, st)

    # -- a run --------------------------------------------------------------------
    def run(self, prompts: Sequence, min_lens: Sequence[int], max_len: int, use_graph: bool = True
            ) -> List[List[Tuple[List[int], float]]]:
        """Hypotheses of every prompt embedding ``(T, hidden)``, best first: (tokens without the stop id,
        sum of log-probabilities)."""
        G, K, R = self.G, self.K, self.R
        lens = [int(np.shape(p)[0]) for p in prompts]
        if len(prompts) != G or len(min_lens) != G:
            raise ValueError(f"{len(prompts)} prompts and {len(min_lens)} minimum lengths for {G} groups")
        if min(lens) < 1 or max(lens) > self.max_prompt or not 1 <= max_len <= self.max_steps:
            raise ValueError(f"prompts of {min(lens)} to {max(lens)} and {max_len} tokens in an engine for {self.max_prompt} and "
                             f"{self.max_steps}")
        # the prompts in one pass through a contiguous cache (freed afterwards), then into pages
        ps = self.cache.page_size
        first = self.m.new_cache(G, -(-max(lens) // ps) * ps)
        last = self.m.forward_batch([D.dev(p) for p in prompts], first)
        self.cache.start_beams(lens, first, K)
        del first
        s = self.state
        s.scores.fill_(-np.inf)
        s.scores[:, 0] = 0.0
        s.counts.zero_()
        s.done.zero_()
        self.min_len.copy_(torch.tensor(list(min_lens), dtype=torch.int32))
        self.cache.bad.zero_()
        st = D.stream()
        rows = torch.zeros((R, self.c.hidden_size), device="cuda")
        rows[::K] = last
        self.head(rows.data_ptr(), R, self.logits.data_ptr(), stream=st)
        self.choose(st)
        self.tokens[0].copy_(s.tokens)
        self.parents[0].copy_(s.parents)
        if use_graph and self.graph is None and max_len > 1:
            # (capture records the step and runs nothing)
            self.graph = Graph()
            self.graph.capture(self.launches)
        steps = 1
        while steps < max_len and not (steps % self.POLL == 0 and bool(s.done.all())):
            if use_graph:
                self.graph.replay()
            else:
                self.launches(D.stream())
            self.tokens[steps].copy_(s.tokens)
            self.parents[steps].copy_(s.parents)
            steps += 1
        if int(self.cache.bad):
            raise RuntimeError("beam search: the paged cache's tables were damaged")
        tok, par = self.tokens[:steps].cpu().numpy(), self.parents[:steps].cpu().numpy()
        scores, counts, done = s.scores.cpu().numpy(), s.counts.cpu().numpy(), s.done.cpu().numpy()
        out = []
        for g in range(G):
            hyps = []
            for k in range(K):
                if not scores[g, k] > -np.inf:
                    continue
                path, at = [], k
                for t in range(steps - 1, -1, -1):
                    path.append(int(tok[t, g, at]))
                    at = int(par[t, g, at])
                path = path[::-1][:int(counts[g, k])]
                hyps.append((path[:-1] if done[g, k] else path, float(scores[g, k])))
            out.append(hyps)
        return out
