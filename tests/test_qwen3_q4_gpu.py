"""The Qwen3 language model with 4-bit weights and cache (Qwen3Lm variant "q4") and its beam search on the GPU.

Logits: against the oracle's basic graph over the values that the weights, head and cache hold, the bar of
tests/test_qwen3_gpu.py (1e-2 of their range). Keys and values that an f16 rounding moves across a code's border move by a
step; at most one rounding in some 250 lies there (a step is over 250 f16 steps of its group's largest values), so the cache's
relative error stays near sqrt(1/250 / 10) / 15 = 0.2%, inside that bar.
Beam search: its tokens and score must equal those of a plain driver that takes the same model's logits, selects with the
float64 oracle and gathers copies of the caches."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, d=512, qh=4, kvh=2, ffn=1024, vocab=2000)


@pytest.fixture(scope="module")
def small(gpu):
    from lokinfer_amd import qwen3 as M

    cfg = M.Qwen3Config(**CFG)
    return M, cfg, M.random_weights(cfg, 3), np.random.default_rng(4).integers(0, cfg.vocab, 41)


def rel(a, b):
    return np.abs(a - b).max() / np.abs(b).max()


@pytest.mark.parametrize("group", [32, 128])
def test_prefill_and_decode(small, group):
    from oracle import q4 as O
    from oracle import qwen3 as Q

    M, cfg, sd, ids = small
    lm = M.Qwen3Lm(sd, cfg, variant="q4", group=group)
    orc = O.oracle_lm(sd, cfg, Q.Ops(np.float32), 96, group)
    kv = lm.kv_cache(60)
    assert kv.shape == (2, 1, 2, 2, 72 * 64)
    dummy = np.zeros((1, cfg.d), np.float16)
    got, ref = lm(ids, dummy, 0, kv), orc(ids, dummy, 0)
    assert rel(got, ref) <= 1e-2, rel(got, ref)
    for pos in range(41, 47):
        tok = int(np.argmax(ref))
        got, ref = lm([tok], dummy, pos, kv), orc([tok], dummy, pos)
        assert rel(got, ref) <= 1e-2, (pos, rel(got, ref))


def test_chunks_graphs_and_sequences_agree(small):
    M, cfg, sd, ids = small
    dummy = np.zeros((1, cfg.d), np.float16)
    graph, eager = M.Qwen3Lm(sd, cfg, variant="q4"), M.Qwen3Lm(sd, cfg, variant="q4", graph=False)
    none = np.zeros((0, cfg.d), np.float16)
    t1 = M.transcribe(graph, ids, none, 12, stop_at_eos=False)
    assert t1 == M.transcribe(eager, ids, none, 12, stop_at_eos=False) and len(t1) == 12
    one, two = graph.kv_cache(64), graph.kv_cache(64)
    whole = graph(ids, dummy, 0, one)
    graph(ids[:20], dummy, 0, two)
    assert rel(graph(ids[20:], dummy, 20, two), whole) <= 1e-2
    # three sequences a step: each as it is alone, to the roundings of another row count
    kv = graph.kv_cache(64, 3)
    kv.t.copy_(one.t.expand_as(kv.t))
    toks = [5, 900, 1999]
    logits = graph.run(toks, dummy, 41, kv, seqs=3)[0].numpy()
    for i, tok in enumerate(toks):
        alone = graph.kv_cache(64)
        alone.t.copy_(one.t)
        assert rel(logits[i:i + 1], graph([tok], dummy, 41, alone)) <= 1e-2
    # a prompt of several sequences at once
    both = graph.kv_cache(64, 2)
    again = graph.run(np.concatenate([ids, ids]), dummy, 0, both, seqs=2)[0].numpy()
    assert rel(again, np.concatenate([whole, whole])) <= 1e-2


def plain_beams(M, lm, ids, beams, max_new, eos, penalty):
    from oracle import q4 as O

    kv = lm.kv_cache(len(ids) + max_new, beams)
    dummy = np.zeros((1, lm.cfg.d), np.float16)
    logits = lm.run(ids, dummy, 0, kv)[0].numpy()
    scores, done, hyps = np.zeros(1, np.float32), np.zeros(1, np.int64), [[]]
    for n in range(max_new):
        s, parent, tok, now = O.beam_select(logits, scores, done, beams, eos)
        hyps = [hyps[p] + ([] if done[p] else [int(t)]) for p, t in zip(parent, tok)]
        scores, done = s.astype(np.float32), now
        if n + 1 == max_new or done.all():
            break
        kv.t.copy_(kv.t[:, torch.from_numpy(parent).cuda()].clone())
        logits = lm.run(tok, dummy, len(ids) + n, kv, seqs=beams)[0].numpy()
    best = int(np.argmax(scores / np.array([len(h) for h in hyps], np.float32) ** penalty))
    return hyps[best], float(scores[best])


@pytest.mark.parametrize("beams,max_new,penalty", [(1, 6, 1.0), (2, 1, 1.0), (4, 10, 1.0), (9, 7, 0.0)])
def test_beam_search(small, beams, max_new, penalty):
    M, cfg, sd, ids = small
    lm = M.Qwen3Lm(sd, cfg, variant="q4")
    greedy = M.transcribe(lm, ids, np.zeros((0, cfg.d), np.float16), 6, stop_at_eos=False)
    # ids that the search meets early end some of the beams
    for eos in ((1999,), (greedy[2], greedy[1]), tuple(range(500, 504))):
        got = M.beam_search(lm, ids, np.zeros((0, cfg.d), np.float16), beams, max_new, length_penalty=penalty, eos=eos)
        want = plain_beams(M, lm, ids, beams, max_new, eos, penalty)
        assert got[0] == want[0] and abs(got[1] - want[1]) <= 1e-5 * abs(want[1]), (eos, got, want)
        if beams == 1 and not set(greedy) & set(eos):
            assert got[0] == greedy[:max_new]


def test_beams_that_take_the_audio_token(small, monkeypatch):
    """An audio id among the generated ones is embedded as a row of zeros for every beam that took it."""
    from lokinfer_amd.f16_gpu import PAD_ID
    from lokinfer_amd.runtime import check_device_errors

    M, _, _, ids = small
    cfg = M.Qwen3Config(layers=1, d=256, qh=2, kvh=1, ffn=256, vocab=PAD_ID + 1)
    lm = M.Qwen3Lm(M.random_weights(cfg, 5), cfg, variant="q4")
    select = M.ops.beam_select_f32_gpu

    def pads(*args):
        s, parents, tok, done = select(*args)
        return s, parents, type(tok)(torch.full_like(tok.t, PAD_ID)), done

    monkeypatch.setattr(M.ops, "beam_select_f32_gpu", pads)
    got = M.beam_search(lm, ids, np.zeros((0, cfg.d), np.float16), 3, 4, eos=(1999,))
    check_device_errors()
    assert got[0] == [PAD_ID] * 4 and np.isfinite(got[1])


def test_refusals(small):
    M, cfg, sd, ids = small
    lm = M.Qwen3Lm(sd, cfg, variant="q4")
    opt = M.Qwen3Lm(sd, cfg)
    none = np.zeros((0, cfg.d), np.float16)
    dummy = np.zeros((1, cfg.d), np.float16)
    for bad in (lambda: M.Qwen3Lm(sd, cfg, variant="q5"), lambda: opt.kv_cache(64, 2),
                lambda: M.beam_search(opt, ids, none, 2, 4), lambda: M.beam_search(lm, ids, none, 33, 4),
                lambda: M.beam_search(lm, ids, none, 2, 4, kv=lm.kv_cache(64, 3)),
                lambda: M.beam_search(lm, ids, none, 2, 40, kv=lm.kv_cache(64, 2)),
                lambda: lm.run(ids, dummy, 0, opt.kv_cache(64)), lambda: lm.run(ids, dummy, 30, lm.kv_cache(64)),
                lambda: lm.run(ids, dummy, 0, lm.kv_cache(64), seqs=2),
                lambda: lm.run(ids[:40], dummy, 0, lm.kv_cache(64, 2), seqs=3),
                lambda: opt.run(ids, dummy, 0, opt.kv_cache(64), seqs=2)):
        with pytest.raises(ValueError):
            bad()
