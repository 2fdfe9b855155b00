"""CPU checks of the contexts that the dense layers' calls take, with contexts and streams that are stand-ins."""
import gc
import threading
from types import SimpleNamespace

import pytest

from burn_automata_amd import _abi

layers = pytest.importorskip("burn_automata_amd.layers")


class Stand:
    made = 0
    closed = 0

    def __init__(self, device, stream):
        type(self).made += 1
        self.device, self.stream = device, stream

    def __del__(self):
        type(self).closed += 1


@pytest.fixture
def stand(monkeypatch):
    class Own(Stand):
        made = closed = 0

    monkeypatch.setattr(layers, "Context", Own)
    monkeypatch.setattr(layers, "_raw_stream", lambda device: 1000 + device)
    monkeypatch.setattr(layers, "_CONTEXTS", type(layers._CONTEXTS)())
    if hasattr(layers, "_Own"):
        monkeypatch.setattr(layers._Own, "free", {})
    return Own


def in_thread(f):
    got = []
    t = threading.Thread(target=lambda: got.append(f()))
    t.start()
    t.join()
    gc.collect()
    return got[0]


def test_a_thread_keeps_its_context_and_threads_do_not_share(stand):
    mine = layers.current_context(0)
    assert layers.current_context(0) is mine and layers.current_context(1) is not mine

    def two():
        a = layers.current_context(0)
        return a is layers.current_context(0) and a is not mine

    assert in_thread(two)
    assert stand.made == 3


def test_a_context_outlives_its_thread_and_serves_the_next_one(stand):
    """What a graph has captured stays allocated when the capturing thread ends, and a program of many short threads
    has no more contexts than threads at once."""
    seen = [in_thread(lambda: id(layers.current_context(0))) for _ in range(5)]
    assert stand.closed == 0 and stand.made == 1 and len(set(seen)) == 1
    barrier = threading.Barrier(3)

    def hold():
        ctx = layers.current_context(0)
        barrier.wait(20)
        return id(ctx)

    got = []
    threads = [threading.Thread(target=lambda: got.append(hold())) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(set(got)) == 3 and stand.made == 3 and stand.closed == 0


def test_a_context_on_another_stream_is_refused(stand):
    x = SimpleNamespace(get_device=lambda: 0, device="cuda:0")
    here = SimpleNamespace(device=0, stream=1000)
    assert layers._context(x, here) is here
    with pytest.raises(_abi.InvalidArgument, match="stream 0x7 .* current stream 0x3e8"):
        layers._context(x, SimpleNamespace(device=0, stream=7))
    with pytest.raises(_abi.InvalidArgument, match="device 1"):
        layers._context(x, SimpleNamespace(device=1, stream=1000))
