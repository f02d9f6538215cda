"""GPU: a decode session as generate() itself builds it is no reference cycle.  (A captured graph that only a cycle keeps alive is destroyed whenever Python's cyclic collector
runs, and torch's destructor synchronizes the device: neuspeech1_amd.lib.capture_section.)"""
import gc
import weakref

import pytest
import torch

from neuspeech1_amd.weights import TINY, make_state_dict, synth_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("num_beams", [1, 3])
@pytest.mark.parametrize("how", ["generator dropped", "sessions cleared"])
def test_sessions_are_freed_without_the_collector(dev, num_beams, how):
    from neuspeech1_amd.engine import MegWhisperEngine
    from neuspeech1_amd.generate import Generator
    x, labels = synth_batch(TINY, 2, 1234)
    x, prompt = torch.from_numpy(x).to(dev), torch.from_numpy(labels[:, :4].copy()).to(dev)
    eng = MegWhisperEngine(TINY, make_state_dict(TINY, 42), device=dev)
    gen = Generator(eng)
    gen.adaptive = False
    modes = []
    for _ in range(3):                   # recorded lists, captured graphs, the session's graphs
        gen.generate(x, prompt, num_beams=num_beams, max_new_tokens=20, suppress_tokens=(TINY.eos_id,))
        modes.append(gen.last_loop_mode)
    assert modes[0].startswith("lists") and modes[1:] == ["graphs", "graphs (session)"], modes
    (ws,) = gen._sessions.values()
    held = [weakref.ref(t) for t in ws["t"].values()] + [weakref.ref(g) for pair in ws["graphs"] for g in pair]
    assert len(held) > 10 and all(r() is not None for r in held)
    torch.cuda.synchronize()
    gc.collect()
    gc.disable()
    try:
        del ws
        if how == "generator dropped":
            del gen
        else:
            gen.clear_sessions()
        left = sum(r() is not None for r in held)
    finally:
        gc.enable()
    assert left == 0, left
