"""Beam search of the speech LM over the paged cache against a beam search written out with the
oracle's forward pass (a cache per hypothesis, scores in float64), and against greedy decoding."""

import copy

import numpy as np
import pytest

from conftest import pkg

import oracle.stages as st

pytestmark = pytest.mark.gpu


def _oracle_beam(lm, x0, K, max_len, min_len, alpha):
    """Best-first hypotheses (tokens, score, done): every live one is continued by every token."""
    sts, stops = lm.speech_token_size, 200
    hyps = [([], 0.0, False, lm.body.new_cache(), x0)]
    for _ in range(max_len):
        cand = []
        for i, (toks, score, done, cache, x) in enumerate(hyps):
            if done:
                cand.append((score / max(len(toks), 1) ** alpha, i, 0, score, True))
                continue
            h = lm.body.forward(x, cache)
            z = lm.head(h[-1:]).astype(np.float64)[0]
            lp = z - z.max()
            lp -= np.log(np.exp(lp).sum())
            if len(toks) < min_len:
                lp[sts:sts + stops] = -np.inf
            for v in np.argsort(-lp, kind="stable")[:K]:
                cand.append(((score + lp[v]) / (len(toks) + 1) ** alpha, i, int(v), score + lp[v], False))
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        new = []
        for _, i, v, score, was in cand[:K]:
            toks, _, done, cache, x = hyps[i]
            if was:
                new.append((toks, score, True, cache, x))
            else:
                new.append((toks + [v], score, v >= sts, copy.deepcopy(cache), lm.speech_emb([v])))
        hyps = new
        if all(h[2] for h in hyps):
            break
    return [(t[:-1] if d else t, s) for t, s, d, _, _ in hyps]


def _models(W):
    lm = pkg("models.llm").CosyVoice3LM(pkg("weights").DeviceWeights(W))
    return lm, st.SpeechLM(W, W.meta)


def _prompts(lm, olm, W, sizes, seed):
    rng = np.random.default_rng(seed)
    eop = W.meta["endofprompt_id"]
    a, b = [], []
    for n in sizes:
        text = [eop] + rng.integers(0, 2000, size=n).tolist()
        sp = rng.integers(0, 256, size=int(rng.integers(0, 9))).tolist()
        a.append(lm.prompt_embedding(text, (), sp))
        b.append(olm.prompt_embedding(text, (), sp))
    return a, b


@pytest.mark.parametrize("profile", ["balanced", "f32"])
@pytest.mark.parametrize("beams,alpha,page_size", [(1, 0.0, 16), (4, 0.0, 16), (3, 0.8, 5), (5, 1.0, 1)])
def test_beam_search_matches_the_oracle(small_weights, profile, beams, alpha, page_size):
    """Tokens equal, scores within 1e-5 of their size (the suite's bar for fp32 log-probabilities,
    added up over the tokens)."""
    W = small_weights[profile]
    lm, olm = _models(W)
    sizes = (3, 14, 40)
    prompts, oprompts = _prompts(lm, olm, W, sizes, 5 + beams)
    mins = [4, 9, 0]
    got = lm.generate_beam(prompts, beams, 14, mins, alpha, page_size)
    for b in range(len(sizes)):
        want = _oracle_beam(olm, oprompts[b], beams, 14, mins[b], alpha)
        assert [t for t, _ in got[b]] == [t for t, _ in want], b
        for (_, s), (_, w) in zip(got[b], want):
            assert abs(s - w) <= 1e-5 * max(1.0, abs(w))


def test_one_beam_without_stops_is_greedy_and_graph_is_eager(small_weights):
    W = small_weights["balanced"]
    lm, olm = _models(W)
    prompts, _ = _prompts(lm, olm, W, (6, 30), 3)
    greedy = lm.generate_greedy(prompts, 40).cpu().numpy().tolist()
    one = lm.generate_beam(prompts, 1, 40, 40)
    assert [h[0][0] for h in one] == greedy
    a = lm.generate_beam(prompts, 4, 30, 20)
    b = lm.generate_beam(prompts, 4, 30, 20, use_graph=False)
    c = lm.generate_beam(prompts, 4, 30, 20)
    assert a == b == c
    assert a[0][0][1] >= a[0][-1][1]


def test_engines_share_no_state(small_weights):
    """Two engines' graphs, run in turn, with more prompts than one batch takes and 16-bit caches."""
    import torch
    W = small_weights["balanced"]
    lm, olm = _models(W)
    prompts, _ = _prompts(lm, olm, W, (5, 9, 13, 21, 8, 30, 4, 11, 6), 9)
    alone = [lm.generate_beam([p], 4, 12, 6)[0] for p in prompts]
    together = lm.generate_beam(prompts, 4, 12, 6)
    assert [[t for t, _ in h] for h in together] == [[t for t, _ in h] for h in alone]
    assert lm.generate_beam(prompts[:1], 4, 12, 6)[0] == alone[0]
    for dt in (torch.float16, torch.bfloat16):
        half = lm.generate_beam(prompts[:2], 4, 12, 6, cache_dtype=dt)
        for h, w in zip(half, alone):
            # a cache of 8 (bf16) or 11 bits changes a log-probability by about as much; the best score stays close
            assert abs(h[0][1] - w[0][1]) <= 0.05 * abs(w[0][1])


def test_synthesis_with_beams(small_weights):
    """``SamplingConfig(beams=...)`` reaches synthesis: the tokens are the best hypothesis's."""
    W = small_weights["balanced"]
    tts = pkg("pipeline").CosyVoice3CUDA(W, seed=7)
    rng = np.random.default_rng(4)
    voice = pkg("voice").VoicePack(speech_token=rng.integers(0, 256, size=6),
                                   mel=rng.normal(size=(12, 80)).astype(np.float32),
                                   embedding=rng.normal(size=192).astype(np.float32))
    text, prompt = rng.integers(0, 2000, size=6).tolist(), [W.meta["endofprompt_id"], 5]
    cfg = pkg("models.llm").SamplingConfig(beams=3, max_token_text_ratio=3.0, min_token_text_ratio=2.0)
    out = tts.synthesize_ids([text], prompt, voice, sampling=cfg)
    x = tts.llm.prompt_embedding(text, prompt, voice.speech_token.tolist())
    assert out.speech_tokens[0] == tts.llm.generate_beam([x], 3, 18, 12)[0][0][0]
    assert len(out.audio) == 960 * len(out.speech_tokens[0]) and np.isfinite(out.audio).all()


def test_paged_cache_serves_requests_that_come_and_go():
    """PagedKVCache over two layers: requests of unequal lengths admitted into the places of finished ones; each
    one's attention equals the operator's over a cache that holds nothing else."""
    import torch
    ops = pkg("ops")
    cache = pkg("models.paged").PagedKVCache(2, 2, 64, requests=4, max_len=64, pages=20, page_size=8)
    rng = np.random.default_rng(3)
    cos, sin = (torch.from_numpy(t).cuda() for t in pkg("models.qwen2").rope_tables(64, 64, 1e6))
    rows = [[] for _ in range(4)]
    i32 = dict(dtype=torch.int32, device="cuda")
    for new, rel in (([20, 3, 0, 9], None), ([1, 1, 1, 1], None), ([1, 30, 1, 1], [0, 1, 0, 0]), ([1, 1, 1, 17], [0, 0, 1, 1])):
        step = cache.extend(torch.tensor(new, **i32), sum(new) + 2, None if rel is None else torch.tensor(rel, **i32))
        qkv = torch.from_numpy(rng.normal(size=(2, sum(new) + 2, 6 * 64)).astype(np.float32)).cuda()
        q = [cache.append(layer, qkv[layer], step, 2, cos, sin) for layer in range(2)]
        at = 0
        for b in range(4):
            rows[b] = ([] if rel and rel[b] else rows[b]) + [qkv[:, at + i] for i in range(new[b])]
            at += new[b]
        assert cache.lens.tolist() == [len(r) for r in rows]
        for layer in range(2):
            x = q[layer][:4].contiguous()
            got = cache.attention(layer, x, 0.125)
            for b in range(4):
                n = len(rows[b])
                alone = pkg("models.paged").PagedKVCache(1, 2, 64, requests=1, max_len=64, pages=8, page_size=8)
                if n:
                    s = alone.extend(torch.tensor([n], **i32), n)
                    alone.append(0, torch.stack([r[layer] for r in rows[b]]), s, 2, cos, sin)
                assert torch.equal(got[b:b + 1], alone.attention(0, x[b:b + 1], 0.125)), (layer, b)
    assert int(cache.bad) == 0 and int(cache.free_count) == 20 - sum(-(-len(r) // 8) for r in rows)


def test_beam_refusals(small_weights):
    W = small_weights["balanced"]
    lm, olm = _models(W)
    (p,), _ = _prompts(lm, olm, W, (4,), 1)
    assert lm.generate_beam([], 3, 5) == []
    for kw in (dict(beams=0), dict(beams=33), dict(max_len=0), dict(min_len=[1, 2])):
        with pytest.raises(ValueError):
            lm.generate_beam([p], **{**dict(beams=2, max_len=5), **kw})
    eng = lm.beam_engine(1, 2, 256, 256, 16, None, 0.0)
    with pytest.raises(ValueError):
        eng.run([p, p], [0, 0], 5)
    with pytest.raises(ValueError):
        eng.run([p], [0], 257)


def test_prompts_without_tokens_are_refused(small_weights):
    W = small_weights["balanced"]
    lm, olm = _models(W)
    (p,), _ = _prompts(lm, olm, W, (4,), 1)
    for prompts in ([p[:0]], [p, p[:0]]):
        with pytest.raises(ValueError):
            lm.generate_beam(prompts, 2, 5)
    with pytest.raises(ValueError):
        lm.beam_engine(1, 2, 256, 256, 16, None, 0.0).run([p[:0]], [0], 5)
