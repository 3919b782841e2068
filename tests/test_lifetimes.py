"""What lives on a context is destroyed before it, whatever order the garbage collector takes the python objects in (on the CPU: the library's
calls are recorded)."""
import gc

import pytest

from hologram_b200 import backend as be


class Recorder:
    """Stands in for the library: hands out handles, writes down what is destroyed."""

    def __init__(self):
        self.gone, self.next = [], 100

    def create(self, *args):
        self.next += 1
        args[-1]._obj.value = self.next
        return 0

    def __getattr__(self, name):
        if name.endswith("_create"):
            return self.create
        if name.endswith("_destroy"):
            return lambda handle: self.gone.append((name, handle.value))
        raise AttributeError(name)


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(be, "lib", r)
    yield r
    gc.collect()


def destroyed(r):
    assert len(r.gone) == len(set(r.gone)), "destroyed twice"
    return [name.replace("holo_b200_", "").replace("_destroy", "") for name, _ in r.gone]


def test_closing_the_backend_destroys_what_is_on_it_first(recorder):
    b = be.B200Backend(0)
    kept = [be.DeviceWorkspace(b, 2), be.DevicePool(b), be.DeviceWorkspace(b, 1)]
    b.close()
    assert sorted(destroyed(recorder)[:3]) == ["pool", "workspace", "workspace"] and destroyed(recorder)[3:] == ["ctx"]
    for k in kept:
        k.close()
    b.close()
    assert len(destroyed(recorder)) == 4


def test_closing_a_workspace_destroys_it_once(recorder):
    b = be.B200Backend(0)
    ws = be.DeviceWorkspace(b, 2)
    ws.close()
    ws.close()
    b.close()
    assert destroyed(recorder) == ["workspace", "ctx"]


def test_a_pool_without_a_backend(recorder):
    be.DevicePool().close()
    assert destroyed(recorder) == ["pool"]


@pytest.mark.parametrize("backend_first", [True, False])
def test_a_cycle_of_backend_and_workspaces(recorder, backend_first):
    """Collected together, the backend may be finalised first: its context must not go before what refers to it."""
    b = be.B200Backend(0)
    things = [be.DeviceWorkspace(b, 2), be.DevicePool(b)]
    ring = [b, things] if backend_first else [things, b]
    ring.append(ring)
    b.ring = ring
    del b, things, ring
    gc.collect()
    names = destroyed(recorder)
    assert sorted(names) == ["ctx", "pool", "workspace"] and names[-1] == "ctx"


def test_a_workspace_finalised_after_its_backend_reaches_for_nothing(recorder):
    b = be.B200Backend(0)
    ws = be.DeviceWorkspace(b, 2)
    b._workspaces.clear()          # as the collector leaves it
    b.close()
    assert destroyed(recorder) == ["workspace", "ctx"]
    ws.close()
    assert destroyed(recorder) == ["workspace", "ctx"] and not ws._h
