"""Paged-cache and beam-search operators: the cases they are measured on, their plain forms and their definitions in 64 bits.

Five operators of the decode path.  ``paged_extend`` gives requests their cache pages and their new tokens their slots,
``paged_append`` rotates the fused q/k/v rows and stores keys and values by slot, ``paged_attention`` is one new token's
attention over its pages, ``beam_select`` keeps the best hypotheses of each group, ``paged_reorder`` lets the cache follow
them.  A case's lengths form a ladder from the shortest to the longest, dealt to the requests by the seed.
"""

import importlib
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decode step of a batch of eight utterances: every request gets one more token
        dict(name="extend: decode of 8", op="extend", batch=8, page_size=16, max_blocks=64, lo=64, hi=900, new_lo=1,
             new_hi=1, release_every=0, short=False),
        # a busy server admits prompts into the places of finished requests, next to decoding ones
        dict(name="extend: 512 prompts", op="extend", batch=512, page_size=16, max_blocks=256, lo=0, hi=1500,
             new_lo=1, new_hi=2000, release_every=3, short=False),
        # the speech LM's decode step at batch 8: fp32 rows into an fp32 cache
        dict(name="append: decode of 8", op="append", rows=8, heads=14, kv_heads=2, dim=64, page_size=16, act="f32",
             cache="f32", pages=512, positions=2048, skip_every=0),
        # packed prompts of a larger model, 16-bit rows and cache
        dict(name="append: 16384 prompt rows", op="append", rows=16384, heads=32, kv_heads=8, dim=128, page_size=16,
             act="bf16", cache="bf16", pages=1200, positions=4096, skip_every=97),
        # one utterance alone, about ten seconds of speech: latency
        dict(name="attention: one utterance", op="attention", batch=1, heads=14, kv_heads=2, dim=64, page_size=16,
             act="f32", cache="f32", lo=325, hi=325, window=0),
        # 32 utterances of up to 30 s, the batch the decode engine advances together
        dict(name="attention: 32 utterances", op="attention", batch=32, heads=14, kv_heads=2, dim=64, page_size=16,
             act="f32", cache="f32", lo=64, hi=1650, window=0),
        # one very long context, cache kept in bf16, fp32 activations: the split over the length carries it
        dict(name="attention: one long context", op="attention", batch=1, heads=14, kv_heads=2, dim=64, page_size=32,
             act="f32", cache="bf16", lo=38399, hi=38399, window=0),
        # a ragged batch of a larger model, from a fresh request to a long document
        dict(name="attention: 64 ragged, bf16", op="attention", batch=64, heads=32, kv_heads=8, dim=128, page_size=16,
             act="bf16", cache="bf16", lo=1, hi=16384, window=0),
        # four hypotheses of one utterance over the speech vocabulary and its stop ids
        dict(name="beam: 4 of one utterance", op="beam", groups=1, beams=4, vocab=6761, stops=200, act="f32",
             length_penalty=0.0, finished_every=0),
        # eight hypotheses of 32 requests over the text vocabulary, some of them finished
        dict(name="beam: 8 of 32, large vocab", op="beam", groups=32, beams=8, vocab=151936, stops=4, act="f32",
             length_penalty=0.6, finished_every=7),
        # the cache of four hypotheses of one utterance through the LM's 24 layers
        dict(name="reorder: 4 beams", op="reorder", groups=1, beams=4, layers=24, kv_heads=2, dim=64, page_size=16,
             cache="f32", lo=331, hi=331),
        # eight hypotheses each of 32 utterances
        dict(name="reorder: 32 x 8 beams", op="reorder", groups=32, beams=8, layers=24, kv_heads=2, dim=64,
             page_size=16, cache="f32", lo=70, hi=1650),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["extend", "append", "attention", "attention", "beam", "reorder"])
    ps = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 128])
    act, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
    heads_per, kv = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([32, 64, 64, 96, 128])
    if op == "extend":
        batch = _log_int(rng, 1, 700)
        new_hi = rng.choice([1, 1, 3, 200, 1500])
        hi = _log_int(rng, 1, 2000)
        return dict(op=op, batch=batch, page_size=ps, max_blocks=-(-(hi + new_hi) // ps) + rng.randrange(3), lo=0,
                    hi=hi, new_lo=rng.choice([0, 1]), new_hi=new_hi, release_every=rng.choice([0, 2, 5]),
                    short=rng.random() < 0.3)
    if op == "append":
        rows = _log_int(rng, 1, max(1, min(8000, 150000000 // ((heads_per + 2) * kv * dim * SIZE[act]))))
        return dict(op=op, rows=rows, heads=heads_per * kv, kv_heads=kv, dim=dim, page_size=ps, act=act, cache=cache,
                    pages=-(-rows // ps) + rng.randrange(1, 50), positions=_log_int(rng, 64, 8000),
                    skip_every=rng.choice([0, 3, 50]))
    if op == "attention":
        batch = _log_int(rng, 1, 96)
        hi = _log_int(rng, 1, max(1, min(40000, 1000000000 // (batch * 2 * kv * dim * SIZE[cache]))))
        return dict(op=op, batch=batch, heads=heads_per * kv, kv_heads=kv, dim=dim, page_size=ps, act=act, cache=cache,
                    lo=rng.choice([0, 1, max(1, hi // 2)]) if batch > 1 else hi, hi=hi,
                    window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]))
    groups, beams = _log_int(rng, 1, 32), rng.choice([1, 2, 3, 4, 5, 8, 10, 16])
    if op == "beam":
        vocab = _log_int(rng, max(16, beams), max(64, min(152000, 20000000 // (groups * beams))))
        return dict(op=op, groups=groups, beams=beams, vocab=vocab, stops=rng.choice([0, 1, 3, vocab // 10]), act=act,
                    length_penalty=rng.choice([0.0, 0.5, 1.0]), finished_every=rng.choice([0, 3, 7]))
    hi, beams, kv = _log_int(rng, 1, 1000), min(beams, 8), min(kv, 4)
    layers = max(n for n in (1, 2, 7, 24) if n == 1 or n * groups * beams * kv * dim * ps < 60000000)
    return dict(op=op, groups=groups, beams=beams, layers=rng.choice([1, layers]), kv_heads=kv, dim=dim,
                page_size=ps, cache=cache, lo=rng.randrange(hi + 1) if groups > 1 else hi, hi=hi)


def _ladder(lo, hi, n):
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _visible(case):
    """Keys that each request's token attends to."""
    w = case["window"]
    return [min(x, w) if w else x for x in _ladder(case["lo"], case["hi"], case["batch"])]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _dealt(values, g):
    v = torch.tensor(values, dtype=torch.int32, device="cuda")
    return v[torch.randperm(len(values), generator=g, device="cuda")].contiguous()


def _perm(n, g):
    return torch.randperm(n, generator=g, device="cuda").to(torch.int32)


def _randn(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype) if math.prod(shape) < 1 << 28 \
        else torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op, ps = case["op"], case.get("page_size")
    if op == "extend":
        B, MB = case["batch"], case["max_blocks"]
        lens = _dealt(_ladder(case["lo"], case["hi"], B), g)
        new = torch.randint(case["new_lo"], case["new_hi"] + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        held = (lens + ps - 1) // ps
        first = torch.cumsum(held, 0) - held
        used = int(held.sum())
        room = B * (-(-case["new_hi"] // ps) + 1)
        P = used + (room // 4 + 1 if case["short"] else room)
        ids = _perm(P, g)
        col = torch.arange(MB, device="cuda", dtype=torch.int32)
        tables = torch.where(col < held[:, None], ids[(first[:, None] + col).clamp_(max=P - 1).long()], -1)
        free = torch.full((P,), -1, dtype=torch.int32, device="cuda")
        free[:P - used] = ids[used:]
        every = case["release_every"]
        release = (_perm(B, g) % every == 0).to(torch.int32) if every else None
        s.update(lens=lens, new=new, tables=tables.to(torch.int32).contiguous(), free=free,
                 count=torch.tensor([P - used], dtype=torch.int32, device="cuda"), release=release,
                 tokens=B * case["new_hi"])
    elif op == "append":
        R, H, Hk, D, P = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["pages"]
        slots = torch.randperm(P * ps, generator=g, device="cuda")[:R].contiguous()
        if case["skip_every"]:
            slots[::case["skip_every"]] = -1
        pos = torch.randint(0, case["positions"], (R,), generator=g, device="cuda", dtype=torch.int32)
        inv = 1e6 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        ang = torch.arange(case["positions"], device="cuda", dtype=torch.float64)[:, None] * inv
        ang = torch.cat([ang, ang], 1)
        pools = [_randn((P + 1, Hk, ps, D), g, DTYPE[case["cache"]]) for _ in range(2)]  # the last page: rows not stored
        s.update(qkv=_randn((R, (H + 2 * Hk) * D), g, DTYPE[case["act"]]), slots=slots, pos=pos,
                 cos=ang.cos().float().contiguous(), sin=ang.sin().float().contiguous(), pools=pools,
                 k_pages=pools[0][:P], v_pages=pools[1][:P])
    elif op == "attention":
        B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        lens = _dealt(_ladder(case["lo"], case["hi"], B), g)
        held = (lens + ps - 1) // ps
        MB = max(1, -(-case["hi"] // ps))
        P = int(held.sum()) + 3
        first = torch.cumsum(held, 0) - held
        ids = _perm(P, g)
        col = torch.arange(MB, device="cuda", dtype=torch.int32)
        tables = torch.where(col < held[:, None], ids[(first[:, None] + col).clamp_(max=P - 1).long()], -1)
        dt = DTYPE[case["cache"]]
        k, v = _randn((P, Hk, ps, D), g, dt), _randn((P, Hk, ps, D), g, dt)
        # what lies behind a request's last token is not part of it
        full, rest = lens // ps, lens % ps
        last = torch.where(rest > 0, tables.gather(1, full.clamp(max=MB - 1)[:, None].long())[:, 0], -1)
        behind = torch.zeros((P + 1, ps), dtype=torch.bool, device="cuda")
        behind[torch.where(last >= 0, last, P).long()] = torch.arange(ps, device="cuda") >= rest[:, None]
        for x in (k, v):
            x.masked_fill_(behind[:P, None, :, None], math.nan)
        s.update(q=_randn((B, H, D), g, DTYPE[case["act"]]), k_pages=k, v_pages=v,
                 tables=tables.to(torch.int32).contiguous(), lens=lens, scale=1.0 / math.sqrt(D))
    elif op == "beam":
        G, K, V = case["groups"], case["beams"], case["vocab"]
        logits = _randn((G, K, V), g, torch.float32).mul_(2.5)
        # a few favourites, as a trained model has
        logits += 5 * (torch.rand((G, K, V), generator=g, device="cuda") < 6 / V)
        counts = torch.randint(3, 60, (G, 1), generator=g, device="cuda", dtype=torch.int32).expand(G, K).contiguous()
        done = torch.zeros((G, K), dtype=torch.int32, device="cuda")
        if case["finished_every"] and case["stops"]:
            done = (_perm(G * K, g).view(G, K) % case["finished_every"] == 0).to(torch.int32)
            counts = counts - done * 2
        scores = -3 * counts.float() * (0.8 + 0.4 * torch.rand((G, K), generator=g, device="cuda"))
        s.update(logits=logits.to(DTYPE[case["act"]]), scores=scores, counts=counts, done=done,
                 stop=(V - case["stops"], V) if case["stops"] else None,
                 min_len=torch.randint(0, 40, (G,), generator=g, device="cuda", dtype=torch.int32))
    else:
        G, K, L, Hk, D = (case[k] for k in ("groups", "beams", "layers", "kv_heads", "dim"))
        lens = _dealt(_ladder(case["lo"], case["hi"], G), g)
        MB = case["hi"] // ps + 1
        ids = _perm(G * K * MB, g)  # every beam holds its pages; full ones are shared from now on
        dt = DTYPE[case["cache"]]
        P = G * K * MB
        last = (lens // ps).clamp(max=MB - 1)
        # only the last pages' contents matter: the pools hold these, other entries name pages that are only shared
        tables = ids.view(G * K, MB)
        own_last = tables.gather(1, last.repeat_interleave(K)[:, None].long())[:, 0]
        back = torch.empty(P, dtype=torch.int32, device="cuda")
        order = torch.argsort(own_last.long())
        back.fill_(-1)
        back[own_last[order].long()] = torch.arange(G * K, device="cuda", dtype=torch.int32)
        rest = back < 0
        back[rest] = torch.arange(G * K, P, device="cuda", dtype=torch.int32)
        tables = back[tables.long()].contiguous()
        N = G * K + 1
        pools = [_randn((L, N, Hk, ps, D), g, dt) for _ in range(2)]  # the last page: beams with nothing to copy
        parents = torch.randint(0, K, (G, K), generator=g, device="cuda", dtype=torch.int32)
        s.update(tables=tables, lens=lens.repeat_interleave(K).contiguous(), parents=parents, pools=pools,
                 k_pages=pools[0][:, :N - 1], v_pages=pools[1][:, :N - 1])
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _blocks(n, ps):
    return (n + ps - 1) // ps


def _plain_extend(s):
    lens, new, tables, free, ps, T = s["lens"], s["new"], s["tables"], s["free"], s["page_size"], s["tokens"]
    B, MB = tables.shape
    P = free.shape[0]
    col = torch.arange(MB, device="cuda")
    lens, new = lens.long(), new.clamp(min=0).long()
    rel = s["release"] != 0 if s["release"] is not None else torch.zeros(B, dtype=torch.bool, device="cuda")
    back = torch.where(rel, _blocks(lens, ps), 0)
    at = s["count"].long() + (torch.cumsum(back, 0) - back)[:, None] + col
    give = col < back[:, None]
    stack = torch.cat([free, free[:1]]).scatter_(0, torch.where(give, at, P).clamp(max=P).view(-1), tables.view(-1))[:P]
    have = s["count"].long() + back.sum()
    base = torch.where(rel, 0, lens)
    need = _blocks(base + new, ps) - _blocks(base, ps)
    fits = (torch.cumsum(need, 0) <= have) & (torch.cumsum(new, 0) <= T) & (base + new <= MB * ps)
    served = torch.cumprod(fits.long(), 0)
    n, need = new * served, need * served
    first = _blocks(base, ps)[:, None]
    take = (col >= first) & (col < first + need[:, None])
    src = have - 1 - ((torch.cumsum(need, 0) - need)[:, None] + col - first)
    tables.copy_(torch.where(take, stack[src.clamp(0, P - 1)], tables))
    free.copy_(stack)
    end = torch.cumsum(n, 0)
    row = torch.arange(T, device="cuda")
    seq = torch.searchsorted(end, row, right=True)
    there = seq < B
    b = seq.clamp(max=B - 1)
    pos = torch.where(there, base[b] + row - (end - n)[b], 0)
    slot = tables[b, (pos // ps).clamp(max=MB - 1)].long() * ps + pos % ps
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), end])
    return {"slots": torch.where(there, slot, -1), "seq": torch.where(there, seq, -1).int(), "pos": pos.int(),
            "offsets": offsets.int(), "lens": (base + n).int(), "free_count": (have - need.sum()).int().view(1),
            "tables": tables, "free": free}


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _plain_append(s):
    H, Hk, D, ps, P = s["heads"], s["kv_heads"], s["dim"], s["page_size"], s["pages"]
    qkv = s["qkv"]
    x = qkv.float().view(-1, H + 2 * Hk, D)
    at = s["pos"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k, v = _rotate(x[:, :H], cos, sin), _rotate(x[:, H:H + Hk], cos, sin), x[:, H + Hk:]
    page = torch.where(s["slots"] >= 0, s["slots"] // ps, P)
    off = s["slots"].clamp(min=0) % ps
    for pool, val in zip(s["pools"], (k, v)):
        pool[page, :, off] = val.to(pool.dtype)
    return {"q": q.to(qkv.dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attention(s):
    q, tables, lens, ps, w = s["q"], s["tables"], s["lens"], s["page_size"], s["window"]
    B, H, D = q.shape
    Hk, M = s["kv_heads"], tables.shape[1] * ps
    key = torch.arange(M, device="cuda")
    seen = (key < lens[:, None]) & ((key >= lens[:, None] - w) if w else (key >= 0))
    at = tables.clamp(min=0).long()
    k = s["k_pages"][at].transpose(1, 2).reshape(B, Hk, M, D).float()
    sc = torch.matmul(q.float().view(B, Hk, H // Hk, D) * s["scale"], k.transpose(2, 3))
    del k
    sc = torch.where(seen[:, None, None], sc, -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    v = s["v_pages"][at].transpose(1, 2).reshape(B, Hk, M, D).float()
    v = torch.where(seen[:, None, :, None], v, 0)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1)
    lse = (top + torch.log(total)).view(B, H)
    return {"out": o.view(B, H, D).to(q.dtype), "lse": lse}


def _plain_beam(s):
    # candidates next to one another can be closer than 32 bits tell apart: keys in 64 bits
    x = s["logits"].double()
    G, K, V = x.shape
    tok = torch.arange(V, device="cuda")
    top = x.amax(-1, keepdim=True)
    logp = x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    done, counts = s["done"] != 0, s["counts"]
    if s["stop"] is not None:
        stops = (tok >= s["stop"][0]) & (tok < s["stop"][1])
        early = counts < s["min_len"][:, None]
        logp = torch.where(early[..., None] & stops, -math.inf, logp)
    else:
        stops = torch.zeros(V, dtype=torch.bool, device="cuda")
    cum = s["scores"].double()[..., None] + logp
    # a finished hypothesis stays as it is: one candidate, its first
    cum = torch.where(done[..., None], torch.where(tok == 0, s["scores"].double()[..., None], -math.inf), cum)
    length = torch.where(done, counts, counts + 1).double()
    key = cum / (length ** s["length_penalty"])[..., None]
    best = torch.sort(key.view(G, K * V), descending=True, stable=True)[1][:, :K]
    parent, token = best // V, best % V
    was = done.gather(1, parent)
    token = torch.where(was, 0, token)
    return {"tokens": token, "parents": parent.int(), "scores": cum.view(G, -1).gather(1, best).float(),
            "counts": (counts.gather(1, parent) + (~was).int()).int(),
            "done": (was | stops[token] & ~was).int()}


def _plain_reorder(s):
    tables, lens, ps = s["tables"], s["lens"], s["page_size"]
    G, K = s["parents"].shape
    MB = tables.shape[1]
    L, N = s["pools"][0].shape[:2]
    row = (s["parents"].long() + torch.arange(G, device="cuda")[:, None] * K).view(-1)
    n = lens.view(G, K)[:, :1].expand(G, K).reshape(-1).long()
    full, rest = n // ps, n % ps
    moved = torch.where(torch.arange(MB, device="cuda") < full[:, None], tables[row], tables)
    mine = tables.gather(1, full.clamp(max=MB - 1)[:, None])[:, 0].long()
    copied = torch.arange(ps, device="cuda") < rest[:, None]
    src = torch.where(rest > 0, mine[row], N - 1)
    dst = torch.where(rest > 0, mine, N - 1)
    for pool in s["pools"]:
        pool[:, dst] = torch.where(copied[None, :, None, :, None], pool[:, src], pool[:, dst])
    tables.copy_(moved)
    return {"tables": tables, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

_ops = None


def _own(s):
    global _ops
    if _ops is None:
        _ops = importlib.import_module("cosyvoice3-cpu_b200.ops")
    op = s["op"]
    if op == "extend":
        r = _ops.paged_extend(s["lens"], s["new"], s["tables"], s["free"], s["count"], s["page_size"], s["tokens"],
                              release=s["release"])
        return {"slots": r.slots, "seq": r.seq, "pos": r.pos, "offsets": r.offsets, "lens": r.lens,
                "free_count": r.free_count, "tables": s["tables"], "free": s["free"]}
    if op == "append":
        q = _ops.paged_append(s["qkv"], s["slots"], s["pos"], s["k_pages"], s["v_pages"], s["heads"], s["cos"], s["sin"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if op == "attention":
        o, lse = _ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], scale=s["scale"],
                                      window=s["window"], return_lse=True)
        return {"out": o, "lse": lse}
    if op == "beam":
        r = _ops.beam_select(s["logits"], s["scores"], s["counts"], s["done"], stop=s["stop"], min_len=s["min_len"],
                             length_penalty=s["length_penalty"])
        return {"tokens": r.tokens, "parents": r.parents, "scores": r.scores, "counts": r.counts, "done": r.done}
    _ops.paged_reorder(s["k_pages"], s["v_pages"], s["tables"], s["parents"], s["lens"])
    return {"tables": s["tables"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


_PLAIN = {"extend": _plain_extend, "append": _plain_append, "attention": _plain_attention, "beam": _plain_beam,
          "reorder": _plain_reorder}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op, ps = case["op"], case.get("page_size")
    if op == "extend":
        B, lens = case["batch"], _ladder(case["lo"], case["hi"], case["batch"])
        tokens = B * (case["new_lo"] + case["new_hi"]) / 2 * (0.5 if case["short"] else 1)
        freed = sum(-(-n // ps) for n in lens) / case["release_every"] if case["release_every"] else 0
        # lengths in and out, page ids moved between the stack and the tables, three numbers a row
        return {"bytes": 20 * B + 8 * (tokens / ps + freed) + 16 * B * case["new_hi"], "flops": 0}
    if op == "append":
        R, H, Hk, D = case["rows"], case["heads"], case["kv_heads"], case["dim"]
        a, c = SIZE[case["act"]], SIZE[case["cache"]]
        tab = min(R, case["positions"]) * 2 * D * 4
        return {"bytes": R * (H + 2 * Hk) * D * a + R * H * D * a + 2 * R * Hk * D * c + tab + 12 * R,
                "flops": 3 * R * (H + Hk) * D}
    if op == "attention":
        H, Hk, D, n = case["heads"], case["kv_heads"], case["dim"], sum(_visible(case))
        return {"bytes": 2 * n * Hk * D * SIZE[case["cache"]] + 2 * case["batch"] * H * D * SIZE[case["act"]] + 4 * n // ps,
                "flops": 4 * n * H * D}
    if op == "beam":
        n = case["groups"] * case["beams"]
        return {"bytes": n * (case["vocab"] * SIZE[case["act"]] + 40), "flops": 4 * n * case["vocab"]}
    # three beams of four follow another one, more or less: what is copied is read and written once
    lens = _ladder(case["lo"], case["hi"], case["groups"])
    K = case["beams"]
    moved = K - 1
    rows = sum(n % ps for n in lens) * moved
    return {"bytes": 2 * rows * case["layers"] * 2 * case["kv_heads"] * case["dim"] * SIZE[case["cache"]]
            + sum(8 * moved * (n // ps) for n in lens) + 8 * K * len(lens), "flops": 0}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    if op in ("extend", "reorder"):
        return None  # page numbers and copies
    s = prepare(case, seed)
    if op == "append":
        H, Hk, D, ps = s["heads"], s["kv_heads"], s["dim"], s["page_size"]
        rows = s["qkv"].double()
        where = s["pos"].long()
        c, n = s["cos"].double()[where], s["sin"].double()[where]
        keys, values = s["k_pages"].double(), s["v_pages"].double()
        kept = torch.nonzero(s["slots"] >= 0)[:, 0]
        page, off = s["slots"][kept] // ps, s["slots"][kept] % ps
        half, turned = D // 2, []
        for h in range(H + Hk):
            x = rows[:, h * D:(h + 1) * D]
            y = torch.empty_like(x)
            y[:, :half] = x[:, :half] * c[:, :half] - x[:, half:] * n[:, :half]
            y[:, half:] = x[:, half:] * c[:, half:] + x[:, :half] * n[:, half:]
            turned.append(y)
        for h in range(Hk):
            keys[page, h, off] = turned[H + h][kept]
            values[page, h, off] = rows[kept, (H + Hk + h) * D:(H + Hk + h + 1) * D]
        return {"q": torch.stack(turned[:H], 1), "k_pages": keys, "v_pages": values}
    if op == "attention":
        ps, w = s["page_size"], s["window"]
        B, H, D = s["q"].shape
        group = H // s["kv_heads"]
        out = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
        lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            first = max(0, n - w) if w else 0
            if n == first:
                continue
            pages = s["tables"][b, :-(-n // ps)].long()
            k = s["k_pages"][pages].permute(1, 0, 2, 3).flatten(1, 2)[:, first:n].double()
            v = s["v_pages"][pages].permute(1, 0, 2, 3).flatten(1, 2)[:, first:n].double()
            for h in range(s["kv_heads"]):
                mine = slice(h * group, (h + 1) * group)
                a = s["scale"] * (s["q"][b, mine].double() @ k[h].T)
                lse[b, mine] = torch.logsumexp(a, 1)
                out[b, mine] = torch.softmax(a, 1) @ v[h]
        return {"out": out, "lse": lse}
    G, K, V = s["logits"].shape
    scores = torch.empty((G, K), dtype=torch.float64, device="cuda")
    for gi in range(G):
        found = []
        for k in range(K):
            have, n = float(s["scores"][gi, k]), int(s["counts"][gi, k])
            if int(s["done"][gi, k]):
                found.append((have / n ** s["length_penalty"], have))
                continue
            x = s["logits"][gi, k].double()
            x = x - torch.logsumexp(x, 0)
            if s["stop"] is not None and n < int(s["min_len"][gi]):
                x[s["stop"][0]:s["stop"][1]] = -math.inf
            found += [((have + v) / (n + 1) ** s["length_penalty"], have + v) for v in torch.topk(x, min(K, V))[0].tolist()]
        found.sort(key=lambda t: -t[0])
        scores[gi] = torch.tensor([v for _, v in found[:K]], dtype=torch.float64)
    return {"tokens": None, "parents": None, "scores": scores, "counts": None, "done": None}
