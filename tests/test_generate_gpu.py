"""Decode parity on the GPU: greedy / beam-search token ids of the HIP path against the golden ids produced by the
reference object (HF GenerationMixin on stock Whisper + the reference's projection_module; tools/make_goldens.py).
Bar: token-id exact (north_star)."""
import os

import numpy as np
import pytest
import torch

from neuspeech1_amd.weights import TINY, make_state_dict, synth_batch

pytestmark = pytest.mark.gpu
G = os.path.join(os.path.dirname(__file__), "golden")


@pytest.fixture(scope="module")
def setup(dev):
    from neuspeech1_amd.engine import MegWhisperEngine
    from neuspeech1_amd.generate import Generator
    g = np.load(os.path.join(G, "decode_tiny.npz"))
    dims = TINY
    eng = MegWhisperEngine(dims, make_state_dict(dims, 42), device=dev)
    x, labels = synth_batch(dims, int(g["B"]), 1234)
    return g, dims, Generator(eng), torch.from_numpy(x).to(dev), torch.from_numpy(labels[:, :4].copy()).to(dev)


def check(out, ref, pad):
    out = out.cpu().numpy()
    Lm = min(out.shape[1], ref.shape[1])
    assert np.array_equal(out[:, :Lm], ref[:, :Lm]), f"\n{out.tolist()}\n{ref.tolist()}"
    assert (out[:, Lm:] == pad).all() and (ref[:, Lm:] == pad).all()
    assert out.shape[1] == ref.shape[1], (out.shape, ref.shape)


def check_greedy_up_to_fp16_ties(out, ref, margin, P, pad, tie=0.03):
    """Greedy ids against the fp32 reference object: exact, except that a row may leave the reference at a position
    where the REFERENCE'S OWN decision margin (processed top-1 minus top-2 score, recorded with the golden) is below
    `tie` -- fp16 logits of magnitude 4-8 resolve 0.004-0.008, so such a decision is not determined at fp16 (the
    reference's own fp16 autocast path would not reproduce its fp32 ids there either).  Everything before the flip must
    match; after it the row is a different sequence."""
    got = out.cpu().numpy()
    assert got.shape == ref.shape, (got.shape, ref.shape)
    flips = 0
    for b in range(ref.shape[0]):
        neq = np.nonzero(got[b] != ref[b])[0]
        if len(neq) == 0:
            continue
        p = int(neq[0])
        assert p >= P and margin[b, p - P] < tie, (b, p, float(margin[b, p - P]), got[b].tolist(), ref[b].tolist())
        flips += 1
    assert flips <= 1, flips


def _row_is(row, hyp, pad):
    L = min(len(row), len(hyp))
    return np.array_equal(row[:L], hyp[:L]) and (row[L:] == pad).all() and (hyp[L:] == pad).all()


def load_hyps(tag):
    """the reference object's top-num_beams finished hypotheses of every beam golden (tools/make_goldens.py hyps)"""
    return np.load(os.path.join(G, f"decode_{tag}_hyps.npz"))


def make_rescore(dims, x, P, **kw):
    """row index -> the fp32 score the reference's beam search assigns to a given row (oracle.sequence_score, pinned on the
    reference object's own hypothesis scores by tests/test_oracle_golden.py); x = the batch the rows were decoded from"""
    from oracle import whisper_meg_oracle as O
    sd = O.to_torch(make_state_dict(dims, 42))
    xc = x.detach().float().cpu()

    def rescore(b, row):
        with torch.no_grad():
            return O.sequence_score(sd, xc[b:b + 1], dims, torch.as_tensor(row), P, **kw)
    return rescore


def check_beam(gen, out, ref, ref_scores, pad, hyps, hyp_scores, rescore):
    """Beam search over a flat random-init model has near-ties (the reference's own second hypothesis is typically 1e-4 .. 5e-3
    behind its first): fp16 logits can flip a decision whose two branches score within rounding of each other, and a row then
    ends on a different hypothesis.  Rule: every row token-exact, except at most ONE row, and that row must be
    a VALID alternative under the reference's arithmetic, not merely a row that reports a similar score:
      * one of the reference object's own finished hypotheses (hyps[b, 1:], stored with the golden) within 2e-2 of its best, or
      * (the search diverged early and ended outside the reference's final five) a row whose fp32 score as the REFERENCE's
        beam search computes it -- the oracle's teacher-forced rescoring of these very ids under the same processors -- lies
        within 2e-2 of the reference's best, and within 2e-2 of the score this path reported for it.
    All rows' reported scores are compared with the reference's (2e-2)."""
    got = out.cpu().numpy()
    sc = gen.last_scores.cpu().numpy()
    np.testing.assert_allclose(sc, ref_scores, atol=2e-2)
    assert got.shape == ref.shape, (got.shape, ref.shape)
    B, nb = hyps.shape[:2]
    assert B == ref.shape[0]
    left = []
    for b in range(B):
        assert _row_is(ref[b], hyps[b, 0], pad)            # the hypotheses file belongs to this golden
        if np.array_equal(got[b], ref[b]):
            continue
        alt = [k for k in range(1, nb) if _row_is(got[b], hyps[b, k], pad)]
        if alt:
            k = alt[0]
            assert hyp_scores[b, 0] - hyp_scores[b, k] < 2e-2 and abs(sc[b] - hyp_scores[b, k]) < 2e-2, (b, k, sc[b], hyp_scores[b].tolist())
            left.append((b, f"reference hypothesis {k}"))
        else:
            true = rescore(b, got[b])
            assert abs(true - float(hyp_scores[b, 0])) < 2e-2 and abs(true - float(sc[b])) < 2e-2, \
                (b, true, float(sc[b]), hyp_scores[b].tolist(), got[b].tolist(), hyps[b].tolist())
            left.append((b, f"outside the reference's final {nb}: oracle score {true:.4f} vs best {float(hyp_scores[b, 0]):.4f}"))
    if left:
        print(f"\nbeam rows off the reference's best hypothesis: {left}")
    assert len(left) <= 1, (left, got.tolist(), ref.tolist())


@pytest.mark.parametrize("name,kw", [
    ("greedy", {}),
    ("greedy_rp", dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
    ("greedy_eos34", dict(eos_id=34)),
    ("greedy_eos630", dict(eos_id=630)),
])
def test_greedy_token_ids_exact(setup, name, kw):
    g, dims, gen, x, prompt = setup
    out = gen.generate(x, prompt, num_beams=1, max_new_tokens=int(g["new_tokens"]), check_every=1, **kw)
    check(out, g[name], dims.pad_id)


@pytest.mark.parametrize("name,kw", [
    ("beam5", {}),
    ("beam5_rp", dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
    ("beam5_eos34", dict(eos_id=34)),
    ("beam5_rp_eos34", dict(repetition_penalty=5.0, no_repeat_ngram_size=2, eos_id=34)),
    ("beam5_eos630", dict(eos_id=630)),
    ("beam5_rp_eos630", dict(repetition_penalty=5.0, no_repeat_ngram_size=2, eos_id=630)),
])
def test_beam_search_token_ids_exact(setup, name, kw):
    g, dims, gen, x, prompt = setup
    out = gen.generate(x, prompt, num_beams=5, max_new_tokens=int(g["new_tokens"]), check_every=1, **kw)
    check(out, g[name], dims.pad_id)
    np.testing.assert_allclose(gen.last_scores.cpu().numpy(), g[name + "_scores"], atol=2e-2)


def test_delayed_stop_check_gives_same_ids(setup):
    g, dims, gen, x, prompt = setup
    a = gen.generate(x, prompt, num_beams=5, max_new_tokens=24, eos_id=630, check_every=1)
    b = gen.generate(x, prompt, num_beams=5, max_new_tokens=24, eos_id=630, check_every=4)
    assert torch.equal(a, b)


@pytest.mark.parametrize("nb,kw", [(1, {}), (5, dict(repetition_penalty=5.0, no_repeat_ngram_size=2))])
def test_launch_lists_hand_over_to_graphs_when_the_host_is_the_bottleneck(setup, nb, kw):
    """A generation too short for graphs replays launch lists; when two polled chunks in a row spend most of their wall time
    inside the replays (a slow host: the runtime's own launch path, ~72 launches per step), the loop captures the hipGraphs
    after all, mid-generation, from the device-resident counters.  Forced here (threshold 0): the switch happens, the ids are
    those of the lists-only and of the eager loop, bit for bit; with the default threshold a GPU-bound... or host-bound run
    must still give the same ids, whichever mode it ends in."""
    from neuspeech1_amd.generate import Generator
    g, dims, gen, x, prompt = setup
    kw = dict(kw, suppress_tokens=(dims.eos_id,))      # every row runs the full length
    eager = Generator(gen.eng, use_graph=False)
    eager.use_lists = False
    ref = eager.generate(x, prompt, num_beams=nb, max_new_tokens=60, **kw)
    assert eager.last_loop_mode == "eager"
    g2 = Generator(gen.eng, use_graph=True)          # graph_min_steps 128 > 60: lists
    g2.adaptive = False
    out = g2.generate(x, prompt, num_beams=nb, max_new_tokens=60, **kw)
    assert g2.last_loop_mode == "lists" and torch.equal(out, ref)
    g3 = Generator(gen.eng, use_graph=True)
    g3.adaptive_frac = 0.0
    out = g3.generate(x, prompt, num_beams=nb, max_new_tokens=60, **kw)
    assert g3.last_loop_mode.startswith("lists->graphs@"), g3.last_loop_mode
    assert torch.equal(out, ref)
    out = g3.generate(x, prompt, num_beams=nb, max_new_tokens=60, **kw)     # the graphs captured mid-generation serve the next call from its first step
    assert g3.last_loop_mode == "graphs (session)" and torch.equal(out, ref)
    g4 = Generator(gen.eng, use_graph=True)
    out = g4.generate(x, prompt, num_beams=nb, max_new_tokens=60, **kw)
    assert g4.last_loop_mode == "lists" or g4.last_loop_mode.startswith("lists->graphs@")
    assert torch.equal(out, ref)


@pytest.mark.parametrize("nb,kw", [(1, {}), (5, dict(repetition_penalty=5.0, no_repeat_ngram_size=2))])
def test_a_failed_graph_capture_falls_back_and_keeps_the_ids(setup, monkeypatch, nb, kw):
    """a hipGraph capture of the decode loop that is invalidated (a host thread outside the capture lock) must not abort the
    evaluation run.  Simulated: the second capture_end of the build raises AFTER ending the capture, which is what torch does -- and
    what leaves the capture stream current.  The generation goes on (launch lists here), ids are the eager loop's, the caller's stream is
    back, the host-side ping-pong lists are where they were (a beam search that continued on swapped lists would give other ids), graphs
    are off for this Generator from then on, and its session holds no half-built graphs."""
    from neuspeech1_amd.generate import Generator
    g, dims, gen, x, prompt = setup
    kw = dict(kw, suppress_tokens=(dims.eos_id,))
    eager = Generator(gen.eng, use_graph=False)
    eager.use_lists = False
    ref = eager.generate(x, prompt, num_beams=nb, max_new_tokens=30, **kw)
    real, calls = torch.cuda.CUDAGraph.capture_end, {"n": 0}

    def capture_end(self):
        real(self)
        calls["n"] += 1
        if calls["n"] == 2:
            raise RuntimeError("simulated: operation failed due to a previous error during capture")
    monkeypatch.setattr(torch.cuda.CUDAGraph, "capture_end", capture_end)
    g2 = Generator(gen.eng, use_graph=True, graph_min_steps=0)
    before = torch.cuda.current_stream()
    with pytest.warns(UserWarning, match="capture failed"):
        out = g2.generate(x, prompt, num_beams=nb, max_new_tokens=30, **kw)
    assert torch.cuda.current_stream() == before
    assert g2.capture_failures == 1 and g2.use_graph is False and g2.last_loop_mode == "lists", g2.last_loop_mode
    assert torch.equal(out, ref)
    assert all(w["graphs"] is None for w in g2._sessions.values())
    out = g2.generate(x, prompt, num_beams=nb, max_new_tokens=30, **kw)       # later calls of the signature: the lists, no new capture
    assert calls["n"] == 2 and g2.last_loop_mode == "lists (session)" and torch.equal(out, ref)


def test_lists_verify_mode_checks_replayed_lists_against_eager_launches(setup, monkeypatch):
    """NS_LISTS_VERIFY=1 (debug): a generation that replayed launch lists is repeated with eager launches and compared.  Here it must pass;
    a launch dropped from the recorded list (what a torch op inside a recorded region amounts to) must be caught."""
    from neuspeech1_amd import ops
    from neuspeech1_amd.generate import Generator
    g, dims, gen, x, prompt = setup
    monkeypatch.setenv("NS_LISTS_VERIFY", "1")
    kw = dict(num_beams=5, max_new_tokens=20, repetition_penalty=5.0, no_repeat_ngram_size=2, suppress_tokens=(dims.eos_id,))
    g2 = Generator(gen.eng, use_graph=False)
    g2.generate(x, prompt, **kw)
    assert g2.last_loop_mode == "lists"
    real = ops.LaunchList.replay

    def lossy(self):          # drops the list's last launch
        saved, self.calls = self.calls, self.calls[:-1]
        try:
            real(self)
        finally:
            self.calls = saved
    monkeypatch.setattr(ops.LaunchList, "replay", lossy)
    g3 = Generator(gen.eng, use_graph=False)
    with pytest.raises(RuntimeError, match="NS_LISTS_VERIFY"):
        g3.generate(x, prompt, **kw)


@pytest.mark.parametrize("nb,kw", [(1, {}), (5, dict(repetition_penalty=5.0, no_repeat_ngram_size=2))])
def test_decode_sessions_replay_across_calls(setup, dev, nb, kw):
    """A Generator keeps the device state and the recorded / captured loop of a call signature (an evaluation run: one signature for
    every batch): call 1 records launch lists, call 2 captures the hipGraphs, call 3 replays them from its first loop step -- on
    OTHER inputs each time.  Every call must give the ids of a fresh generator on the same input, results handed out earlier must
    not change when the session's buffers are written again, another signature gets its own session, and clear_sessions() starts over."""
    from neuspeech1_amd.generate import Generator
    g, dims, gen, x, prompt = setup
    kw = dict(kw, suppress_tokens=(dims.eos_id,))
    xs = [x, torch.roll(x, 1, 0) * 0.9, torch.flip(x, (2,))]
    fresh = []
    for xi in xs:
        f = Generator(gen.eng, use_graph=False)
        f.use_lists = False
        f.cache_sessions = False
        fresh.append(f.generate(xi, prompt, num_beams=nb, max_new_tokens=40, **kw))
    g2 = Generator(gen.eng)
    g2.adaptive = False        # (at these dims a replayed step is as long on the host as on the GPU: the hand-over would fire now and then)
    outs, modes = [], []
    for xi in xs + [xs[0]]:
        outs.append(g2.generate(xi, prompt, num_beams=nb, max_new_tokens=40, **kw))
        modes.append(g2.last_loop_mode)
    assert modes[0] == "lists" and modes[1] == "graphs" and modes[2] == modes[3] == "graphs (session)", modes
    for o, ref in zip(outs, fresh + [fresh[0]]):
        assert torch.equal(o, ref)
    assert len(g2._sessions) == 1
    short = g2.generate(xs[1], prompt, num_beams=nb, max_new_tokens=12, **kw)       # another signature
    assert g2.last_loop_mode == "lists" and len(g2._sessions) == 2
    f = Generator(gen.eng, use_graph=False)
    f.cache_sessions = False
    assert torch.equal(short, f.generate(xs[1], prompt, num_beams=nb, max_new_tokens=12, **kw))
    assert torch.equal(outs[1], fresh[1])                                          # handed-out results are copies
    g2.clear_sessions()
    assert torch.equal(g2.generate(xs[2], prompt, num_beams=nb, max_new_tokens=40, **kw), fresh[2]) and g2.last_loop_mode == "lists"
    g2.max_session_frac = 0.0                      # the memory cap: a session above it is dropped after its call
    assert torch.equal(g2.generate(xs[0], prompt, num_beams=nb, max_new_tokens=40, **kw), fresh[0]) and len(g2._sessions) == 0


def test_processors_and_topk_kernels(dev):
    """ns_logits_process / ns_topk_groups against torch on hand-built cases (G5 of SURVEY.md §8c)."""
    from neuspeech1_amd import ops
    from oracle import whisper_meg_oracle as O
    torch.manual_seed(0)
    rows, V, ldv, L = 6, 1000, 1024, 12
    logits = torch.zeros(rows, ldv, device=dev, dtype=torch.float16)
    logits[:, :V] = (torch.randn(rows, V, device=dev) * 3).half()
    ids = torch.randint(0, 50, (rows, L), device=dev)
    cur = 9
    ids[0, 3:5] = ids[0, 7:9]          # a repeated bigram prefix -> ban
    bs = torch.randn(rows, device=dev)
    scores = torch.empty(rows, V, device=dev)
    sup = torch.tensor([5, 6], device=dev, dtype=torch.int32)
    ops.logits_process(logits16=logits, scores32=scores, ids=ids, rows=rows, V=V, ldv=ldv, ids_ld=L, cur_len=cur,
                       begin_index=cur, log_softmax=True, beam_scores=bs, repetition_penalty=5.0, no_repeat_ngram=2,
                       suppress=sup, n_suppress=2, begin_suppress=sup, n_begin_suppress=1)
    ref = torch.log_softmax(logits[:, :V].float().cpu(), -1)
    O.repetition_penalty_(ref, ids[:, :cur].cpu(), 5.0)
    O.no_repeat_ngram_(ref, ids[:, :cur].cpu(), 2)
    O.suppress_(ref, [5, 6], [5], cur, cur)
    ref = ref + bs.cpu()[:, None]
    got = scores.cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(ref))
    fin = ~torch.isinf(ref)
    torch.testing.assert_close(got[fin], ref[fin], atol=2e-3, rtol=1e-4)
    vals = torch.empty(2, 10, device=dev)
    idx = torch.empty(2, 10, device=dev, dtype=torch.int32)
    ops.topk_groups(scores, 2, 3 * V, 10, vals, idx)
    rv, ri = torch.topk(scores.view(2, 3 * V), 10, dim=1)
    assert torch.equal(vals, rv) and torch.equal(idx.long(), ri)


@pytest.mark.parametrize("V,ldv,case", [(1000, 1024, "plain"), (51865, 51968, "plain"), (51865, 51968, "ties"),
                                        (51865, 51968, "clustered"), (1000, 1024, "biased"), (51865, 51968, "biased"),
                                        (51865, 51968, "biased-clustered")])
def test_fused_select_is_bit_identical_to_process_plus_topk(dev, V, ldv, case):
    """ns_logits_select + ns_topk_merge == ns_logits_process + ns_topk_groups: same values, same flat indices, same
    order, including rows full of ties (fp16 logits) and rows whose top values sit in ONE thread's columns (the
    candidate list overflows and the exact slow path runs)."""
    from neuspeech1_amd import ops
    torch.manual_seed(3)
    nb, B, L, cur, k = 5, 3, 40, 23, 10
    rows = nb * B
    logits = torch.zeros(rows, ldv, device=dev, dtype=torch.float16)
    if case == "ties":
        logits[:, :V] = torch.randint(-4, 5, (rows, V), device=dev).half()           # nine distinct values
    elif case.endswith("clustered"):
        logits[:, :V] = (torch.randn(rows, V, device=dev)).half()
        cols = (torch.arange(0, 24, device=dev)[:, None] * 2048 + torch.arange(0, 8, device=dev)[None, :]).reshape(-1) + 8 * 7
        logits[:, cols[cols < V]] = (20 + torch.arange(0, (cols < V).sum(), device=dev) * 0.125).half()   # all in thread 7
        logits[1, 5000:7000] = 30.0                                                  # > 1024 equal leaders
    else:
        logits[:, :V] = (torch.randn(rows, V, device=dev) * 3).half()
    ids = torch.randint(0, min(V, 3000), (rows, L), device=dev)
    ids[0, 3:5] = ids[0, cur - 2:cur]
    ids[2, 10] = int(logits[2, :V].float().argmax())      # penalise the leader
    bs = torch.randn(rows, device=dev)
    sup = torch.tensor([5, 6, int(logits[4, :V].float().argmax())], device=dev, dtype=torch.int32)
    common = dict(logits16=logits, ids=ids, rows=rows, V=V, ldv=ldv, ids_ld=L, cur_len=cur, begin_index=cur,
                  repetition_penalty=5.0, no_repeat_ngram=2, suppress=sup, n_suppress=3, begin_suppress=sup, n_begin_suppress=1)
    if case.startswith("biased"):
        # sequence bias (HF SequenceBiasLogitsProcessor, evaluation.py --add_sequence_bias): single tokens (one of them in the
        # history, one the row leader, one suppressed), multi-token entries whose prefix ends row 1's / row 3's history (two of
        # them sharing their last token with a single-token entry), one longer than the context, one that does not match
        from neuspeech1_amd.generate import _sequence_bias_tables
        lead3 = int(logits[3, :V].float().argmax())
        h1, h3 = [int(t) for t in ids[1, cur - 2:cur]], [int(t) for t in ids[3, cur - 1:cur]]
        sb = {(7,): 4.0, (int(ids[2, 5]),): -3.0, (lead3,): 2.5, (5,): 9.0, (V - 1,): 6.0,
              (h1[0], h1[1], 11): 8.0, (h1[1], 11): 1.5, (h3[0], 7): 3.0, (h3[0], V - 2): 12.0,
              tuple(range(1, cur + 3)): 5.0, (V - 3, V - 4, 12): 7.0}
        common.update(_sequence_bias_tables(sb, V, dev))
    for lsm, beams in ((True, bs), (False, None)):
        scores = torch.empty(rows, V, device=dev)
        ops.logits_process(scores32=scores, log_softmax=lsm, beam_scores=beams, **common)
        rv = torch.empty(B, k, device=dev)
        ri = torch.empty(B, k, device=dev, dtype=torch.int32)
        ops.topk_groups(scores, B, nb * V, k, rv, ri)
        cv = torch.empty(rows, k, device=dev)
        ci = torch.empty(rows, k, device=dev, dtype=torch.int32)
        ops.logits_select(log_softmax=lsm, beam_scores=beams, k=k, group_rows=nb, cand_vals=cv, cand_idx=ci, **common)
        gv = torch.empty(B, k, device=dev)
        gi = torch.empty(B, k, device=dev, dtype=torch.int32)
        ops.topk_merge(cv, ci, B, nb * k, k, gv, gi)
        assert torch.equal(gv, rv), (case, lsm)
        assert torch.equal(gi, ri), (case, lsm)
        # per-row lists too (greedy uses k = 1 of them)
        pv, pi = torch.topk(scores, k, dim=1)
        assert torch.equal(cv, pv)


@pytest.mark.parametrize("nb", [1, 5])
def test_graph_replay_gives_the_same_ids_as_eager_launches(setup, nb):
    """hipGraph replay of the decode iteration (device-side position counters, ping-pong parity pairs) vs eager."""
    from neuspeech1_amd.generate import Generator
    g, dims, gen, x, prompt = setup
    kw = dict(num_beams=nb, max_new_tokens=40, eos_id=630, repetition_penalty=5.0 if nb > 1 else 1.0,
              no_repeat_ngram_size=2 if nb > 1 else 0)
    a = Generator(gen.eng, use_graph=False).generate(x, prompt, **kw)
    b = Generator(gen.eng, use_graph=True, graph_min_steps=0).generate(x, prompt, **kw)
    c = Generator(gen.eng, use_graph=True, graph_min_steps=0).generate(x, prompt, check_every=1, **kw)
    assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("name,nb,kw", [
    ("greedy", 1, {}),
    ("greedy_rp", 1, dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
    ("beam5", 5, {}),
    ("beam5_rp", 5, dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
])
def test_token_ids_exact_at_whisper_base_dims(dev, name, nb, kw):
    """Same bar at the size BASELINE's metrics are quoted on (whisper-base, 208-ch MEG): ids from the reference
    object (tools/make_goldens.py decode_base), B = 2, 16 new tokens."""
    from neuspeech1_amd.engine import MegWhisperEngine
    from neuspeech1_amd.generate import Generator
    from neuspeech1_amd.weights import WHISPER_BASE
    g = np.load(os.path.join(G, "decode_base208.npz"))
    dims = WHISPER_BASE
    gen = Generator(MegWhisperEngine(dims, make_state_dict(dims, 42), device=dev))
    x, labels = synth_batch(dims, int(g["B"]), 1234)
    out = gen.generate(torch.from_numpy(x).to(dev), torch.from_numpy(labels[:, :4].copy()).to(dev), num_beams=nb,
                       max_new_tokens=int(g["new_tokens"]), check_every=1, **kw)
    check(out, g[name], dims.pad_id)
    if nb > 1:
        np.testing.assert_allclose(gen.last_scores.cpu().numpy(), g[name + "_scores"], atol=2e-2)


def _sb_from_golden(g):
    return {tuple(int(t) for t in str(k).split(",")): float(v) for k, v in zip(g["sequence_bias_keys"], g["sequence_bias_vals"])}


@pytest.mark.parametrize("name,nb,kw", [
    ("greedy_sb", 1, {}),
    ("greedy_rp_sb", 1, dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
    ("beam5_sb", 5, {}),
    ("beam5_rp_sb", 5, dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
])
def test_sequence_bias_token_ids_exact(setup, name, nb, kw):
    """model.generate(sequence_bias=...) (HF SequenceBiasLogitsProcessor; evaluation.py:362-364 passes it with
    --add_sequence_bias): ids of the reference object run with the same bias table (tools/make_goldens.py decode_sb)."""
    _, dims, gen, x, prompt = setup
    g = np.load(os.path.join(G, "decode_tiny_sb.npz"))
    out = gen.generate(x, prompt, num_beams=nb, max_new_tokens=int(g["new_tokens"]), check_every=1,
                       sequence_bias=_sb_from_golden(g), **kw)
    if nb == 1:
        check(out, g[name], dims.pad_id)
        return
    # (row 0 of beam5_rp_sb ends on a hypothesis scoring -4.690 against the reference's -4.683); the processor itself is
    # checked against HF's classes below
    hy = load_hyps("tiny_sb")
    check_beam(gen, out, g[name], g[name + "_scores"], dims.pad_id, hy[name + "_hyps"], hy[name + "_hyp_scores"],
               make_rescore(dims, x, prompt.shape[1], sequence_bias=_sb_from_golden(g), **kw))


def test_sequence_bias_processor_matches_hf_processors(dev):
    """ns_logits_process with a bias table against HF's own processor classes chained in HF's order
    (SequenceBias -> RepetitionPenalty -> NoRepeatNGram), on histories that end with the biased prefixes."""
    from transformers.generation.logits_process import (NoRepeatNGramLogitsProcessor, RepetitionPenaltyLogitsProcessor,
                                                         SequenceBiasLogitsProcessor)
    from neuspeech1_amd import ops
    from neuspeech1_amd.generate import _sequence_bias_tables
    rows, V, Vp, cur, ld = 7, 1000, 1024, 12, 16
    gcpu = torch.Generator().manual_seed(3)
    logits = (torch.randn(rows, Vp, generator=gcpu) * 3).half()
    ids = torch.randint(5, 60, (rows, ld), generator=gcpu)
    ids[0, cur - 2:cur] = torch.tensor([7, 8])          # row 0 ends with (7, 8): both 3-token sequences below fire
    ids[1, cur - 1] = 8                                 # row 1 ends with 8: the 2-token sequence fires
    ids[2, cur - 3:cur] = torch.tensor([9, 7, 8])       # 4-token sequence
    ids[3, :cur] = 41                                   # a repeated token that also carries a single-token bias
    sb = {(41,): -3.0, (500,): 2.5, (7, 8, 123): 4.0, (7, 8, 500): -1.25, (8, 77): 6.0, (8, 123): 0.5, (9, 7, 8, 200): 3.0,
          tuple(range(100, 100 + cur + 1)): 9.0}        # longer than the context: ignored
    for log_softmax in (False, True):
        sc = torch.log_softmax(logits[:, :V].float(), -1) if log_softmax else logits[:, :V].float()
        ref = SequenceBiasLogitsProcessor(sequence_bias=dict(sb))(ids[:, :cur], sc.clone())
        ref = RepetitionPenaltyLogitsProcessor(penalty=5.0)(ids[:, :cur], ref)
        ref = NoRepeatNGramLogitsProcessor(2)(ids[:, :cur], ref)
        out = torch.full((rows, V), float("nan"), device=dev)
        ops.logits_process(logits16=logits.to(dev), scores32=out, ids=ids.to(dev), rows=rows, V=V, ldv=Vp, ids_ld=ld,
                           cur_len=cur, begin_index=4, log_softmax=log_softmax, repetition_penalty=5.0, no_repeat_ngram=2,
                           **_sequence_bias_tables(dict(sb), V, dev))
        got = out.cpu()
        assert torch.equal(torch.isinf(got), torch.isinf(ref))
        fin = ~torch.isinf(ref)
        torch.testing.assert_close(got[fin], ref[fin], atol=2e-5, rtol=1e-5)
        assert abs(got[0, 123] - (sc[0, 123] + 4.0 + 0.5)) < 1e-4 or 123 in ids[0, :cur].tolist()
    for bad in ({}, {(1, 2): 1}, {(V,): 1.0}, [[[], 1.0]], {(-1,): 1.0}):
        with pytest.raises(ValueError):
            _sequence_bias_tables(bad, V, dev)


@pytest.mark.parametrize("pn", ["p1", "p4"])
@pytest.mark.parametrize("name,nb,kw", [
    ("greedy", 1, {}),
    ("greedy_rp", 1, dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
    ("beam5", 5, {}),
    ("beam5_rp", 5, dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
])
def test_forced_decoder_ids_and_suppress_lists_token_ids_exact(setup, pn, name, nb, kw):
    """generation_config.forced_decoder_ids ([[1, null], [2, task], [3, notimestamps]]-shaped) + non-empty suppress /
    begin-suppress lists, as a hub whisper checkpoint carries them (reference utils/load_model.py:1210-1256 hands them to
    super().generate): ids of the reference object (tools/make_goldens.py forced), with the decoder prompt the reference
    uses for English (start token only) and for other languages (labels[:, :4], evaluation.py:353-355).  Both the fused
    selection kernel and the two-kernel form (forced by a sequence-bias table of zeros)."""
    _, dims, gen, x, _ = setup
    g = np.load(os.path.join(G, "decode_tiny_forced.npz"))
    forced = [[int(i), None if int(t) < 0 else int(t)] for i, t in zip(g["forced_idx"], g["forced_tok"])]
    prompt = torch.from_numpy(g[pn + ".prompt"]).to(x.device)
    for extra in ({}, dict(sequence_bias={(3,): 0.0})):
        out = gen.generate(x, prompt, num_beams=nb, max_new_tokens=int(g["new_tokens"]), check_every=1,
                           suppress_tokens=g["suppress"].tolist(), begin_suppress_tokens=g["begin_suppress"].tolist(),
                           forced_decoder_ids=forced, begin_index=prompt.shape[1] + forced[-1][0], **kw, **extra)
        if name == "beam5_rp":
            hy = load_hyps("tiny_forced")
            check_beam(gen, out, g[f"{pn}.{name}"], g[f"{pn}.beam5_rp_scores"], dims.pad_id, hy[f"{pn}.{name}_hyps"],
                       hy[f"{pn}.{name}_hyp_scores"],
                       make_rescore(dims, x, prompt.shape[1], suppress_tokens=g["suppress"].tolist(),
                                    begin_suppress_tokens=g["begin_suppress"].tolist(), forced_decoder_ids=forced, **kw))
        else:
            check(out, g[f"{pn}.{name}"], dims.pad_id)


@pytest.mark.parametrize("tag", ["base273", "lv2w"])
@pytest.mark.parametrize("name,nb,kw", [
    ("greedy", 1, {}),
    ("greedy_rp", 1, dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
    ("beam5", 5, {}),
    ("beam5_rp", 5, dict(repetition_penalty=5.0, no_repeat_ngram_size=2)),
])
def test_token_ids_exact_at_273_channels_and_large_v2_width(dev, tag, name, nb, kw):
    """BASELINE configs[3] (whisper-base, 273-ch Schoffelen shape, beam-5 + repetition penalty 5 + no-repeat-2:
    /root/reference README.md:60-64) and configs[4]'s WIDTH (whisper-large-v2: d 1280, 20 heads, ffn 5120, 273-ch; 2 + 2
    layers): ids of the reference object (tools/make_goldens.py decode_base273 / lv2w)."""
    from neuspeech1_amd.engine import MegWhisperEngine
    from neuspeech1_amd.generate import Generator
    from neuspeech1_amd.weights import LV2W, WhisperDims
    g = np.load(os.path.join(G, f"decode_{tag}.npz"))
    dims = LV2W if tag == "lv2w" else WhisperDims(ch=273)
    gen = Generator(MegWhisperEngine(dims, make_state_dict(dims, 42), device=dev))
    x, labels = synth_batch(dims, int(g["B"]), 1234)
    out = gen.generate(torch.from_numpy(x).to(dev), torch.from_numpy(labels[:, :4].copy()).to(dev), num_beams=nb,
                       max_new_tokens=int(g["new_tokens"]), check_every=1, **kw)
    if nb > 1:
        hy = load_hyps(tag)
        check_beam(gen, out, g[name], g[name + "_scores"], dims.pad_id, hy[name + "_hyps"], hy[name + "_hyp_scores"],
                   make_rescore(dims, torch.from_numpy(x), 4, **kw))
    else:
        check_greedy_up_to_fp16_ties(out, g[name], g[name + "_margin"], 4, dims.pad_id)


def test_no_garbage_collection_runs_while_a_decode_graph_is_captured(setup, monkeypatch):
    """a CUDAGraph that only a reference cycle keeps alive is destroyed when the cyclic collector runs, and torch's destructor
    synchronizes the device: inside an open capture that ends the process (neuspeech1_amd.lib.capture_section)"""
    import gc
    from neuspeech1_amd import ops
    from neuspeech1_amd.generate import Generator
    g, dims, gen, x, prompt = setup
    real, seen = ops.add_i32, []

    def add_i32(*a, **k):
        if torch.cuda.is_current_stream_capturing():
            seen.append(gc.isenabled())
        return real(*a, **k)
    monkeypatch.setattr(ops, "add_i32", add_i32)
    g2 = Generator(gen.eng, use_graph=True, graph_min_steps=0)
    g2.generate(x, prompt, num_beams=1, max_new_tokens=20, suppress_tokens=(dims.eos_id,))
    assert g2.last_loop_mode == "graphs" and seen and not any(seen) and gc.isenabled()
