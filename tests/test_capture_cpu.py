"""CPU: nothing that a garbage collection may destroy is destroyed while a hipGraph capture is open.  (torch's ~CUDAGraph synchronizes the
device on ROCm; inside a capture that fails, in a destructor, and ends the process.)"""
import contextlib
import gc
import types
import weakref

import pytest
import torch


class _Graph:
    """stands for a captured graph: notes whether it was destroyed while a capture was open"""
    capturing = False
    destroyed_inside = 0

    def __del__(self):
        if _Graph.capturing:
            _Graph.destroyed_inside += 1


def _garbage_cycle():
    a, b = {}, {}
    a["other"], b["other"], a["graph"] = b, a, _Graph()


@contextlib.contextmanager
def _fake_capture(*a, **k):
    _Graph.capturing = True
    try:
        yield
    finally:
        _Graph.capturing = False


def _allocate_much():
    keep = [[i] for i in range(200000)]     # container allocations: what starts the collector
    return len(keep)


@pytest.fixture(autouse=True)
def _reset():
    gc.collect()
    _Graph.destroyed_inside, _Graph.capturing = 0, False
    yield
    assert gc.isenabled()


def test_the_fake_graph_is_destroyed_by_the_collector_alone():
    _garbage_cycle()
    with _fake_capture():
        _allocate_much()
    assert _Graph.destroyed_inside == 1


def test_capture_section_keeps_the_collector_off_and_nests():
    from neuspeech1_amd import lib
    _garbage_cycle()
    with lib.capture_section():
        with _fake_capture():
            _allocate_much()
        with lib.capture_section():
            assert not gc.isenabled()
        assert not gc.isenabled()
    assert _Graph.destroyed_inside == 0 and gc.isenabled()
    with pytest.raises(RuntimeError):
        with lib.capture_section():
            raise RuntimeError("a capture that failed")
    assert gc.isenabled()
    gc.disable()
    try:
        with lib.capture_section():
            pass
        assert not gc.isenabled()           # the caller's own setting comes back
    finally:
        gc.enable()


def test_a_training_step_capture_destroys_no_graph(monkeypatch):
    from neuspeech1_amd import engine as E
    monkeypatch.setattr(torch.cuda, "CUDAGraph", _Graph)
    monkeypatch.setattr(torch.cuda, "graph", _fake_capture)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "graph_pool_handle", lambda: None)
    me = types.SimpleNamespace(_alloc_enc=lambda B, train: {"xin": torch.zeros(1)}, _graph_graveyard=[], _b={}, zero_grad=lambda: None,
                               forward=lambda *a, **k: _allocate_much(), backward=lambda cut: _allocate_much(), optimizer_step=_allocate_much)
    _garbage_cycle()
    out = E.MegWhisperEngine._capture_step(me, torch.zeros(2, 3, 4), torch.zeros(2, 5, dtype=torch.int64), False)
    assert len(out["segs"]) == 1 and _Graph.destroyed_inside == 0


def test_recorded_lists_do_not_make_their_session_a_cycle():
    """a decode session as the generation loop builds it: dropped, it is freed at once, its graphs with it"""
    import inspect
    from neuspeech1_amd import generate, ops
    assert "gt.keep = ws " not in inspect.getsource(generate)

    class Session(dict):
        pass
    ws = Session(t={"x": torch.zeros(1)}, sb={}, graphs=[_Graph()], lists=None, calls=0)
    lst = ops.LaunchList()
    lst.keep = (ws["t"], ws["sb"])
    ws["lists"] = [(lst, lst)]
    ref = weakref.ref(ws)
    gc.disable()
    try:
        del ws, lst
        assert ref() is None
    finally:
        gc.enable()
