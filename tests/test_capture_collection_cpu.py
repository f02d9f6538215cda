"""CPU: a garbage collection that another thread has begun before a capture opens does not destroy anything inside it either.  (`gc.disable()` keeps collections from starting; one that
runs goes on, and whenever a finalizer of it lets go of the interpreter lock the capturing thread may get ahead of it.)"""
import contextlib
import gc
import threading
import time

import pytest


class _Graph:
    """stands for a captured graph: notes whether it was destroyed while a capture was open"""
    capturing = False
    destroyed = 0
    destroyed_inside = 0

    def __del__(self):
        _Graph.destroyed += 1
        if _Graph.capturing:
            _Graph.destroyed_inside += 1


class _Slow:
    """a finalizer that lets go of the interpreter lock for a while, as closing a file or freeing device memory does"""
    begun = None

    def __del__(self):
        _Slow.begun.set()
        time.sleep(0.4)


@contextlib.contextmanager
def _fake_capture():
    _Graph.capturing = True
    try:
        yield
    finally:
        _Graph.capturing = False


def _garbage_cycle():
    a, b = {}, {}
    a["other"], b["other"] = b, a
    a["slow"] = _Slow()
    a["graph"] = _Graph()


@pytest.fixture(autouse=True)
def _reset():
    gc.collect()
    _Graph.capturing, _Graph.destroyed, _Graph.destroyed_inside = False, 0, 0
    _Slow.begun = threading.Event()
    yield
    assert gc.isenabled()


def _collect_by_allocating():
    keep = []
    while not _Slow.begun.is_set():
        keep.append([len(keep)])
        if len(keep) > 5_000_000:
            return


@pytest.mark.parametrize("how", [gc.collect, _collect_by_allocating], ids=["collect", "allocate"])
def test_a_collection_that_another_thread_has_begun_ends_before_the_capture_opens(how):
    from neuspeech1_amd import lib
    _garbage_cycle()
    t = threading.Thread(target=how)
    t.start()
    assert _Slow.begun.wait(30)
    with lib.capture_section():
        with _fake_capture():
            time.sleep(0.8)
    t.join()
    assert _Graph.destroyed == 1 and _Graph.destroyed_inside == 0


def test_the_collecting_thread_may_need_the_capture_lock():
    """a finalizer that takes the lock (the feed's GPU calls do) is let through before the capture"""
    from neuspeech1_amd import lib

    class Needs:
        got = False

        def __del__(self):
            _Slow.begun.set()
            time.sleep(0.2)
            with lib.GPU_CAPTURE_LOCK:
                Needs.got = not _Graph.capturing
    a = {"needs": Needs()}
    a["self"] = a
    del a
    t = threading.Thread(target=gc.collect)
    t.start()
    assert _Slow.begun.wait(30)
    with lib.capture_section(), _fake_capture():
        time.sleep(0.1)
    t.join(30)
    assert not t.is_alive() and Needs.got


def test_a_capture_inside_a_finalizer_is_refused_and_does_not_hang(monkeypatch):
    from neuspeech1_amd import lib
    monkeypatch.setattr(lib, "COLLECTION_WAIT_S", 0.05)
    seen = []

    class Captures:
        def __del__(self):
            try:
                with lib.capture_section():
                    seen.append("captured")
            except lib.NeuSpeechHipError as e:
                seen.append(str(e))
    a = {"x": Captures()}
    a["self"] = a
    del a
    gc.collect()
    assert len(seen) == 1 and "collection" in seen[0]
    assert lib.GPU_CAPTURE_LOCK.acquire(blocking=False)
    lib.GPU_CAPTURE_LOCK.release()
    with lib.capture_section():
        pass


def test_sections_of_several_threads_keep_the_collector_off():
    from neuspeech1_amd import lib
    off = []

    def work():
        for _ in range(50):
            with lib.capture_section():
                off.append(gc.isenabled())
                time.sleep(0.0005)
                off.append(gc.isenabled())
    ts = [threading.Thread(target=work) for _ in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert len(off) == 400 and not any(off) and gc.isenabled()
