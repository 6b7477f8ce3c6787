"""A capture holds the garbage collector off, and puts it back whatever happens (``torch.cuda.graph`` replaced: no GPU)."""
import contextlib
import gc

import pytest
import torch

from transformerengine_b200 import graph


@pytest.mark.parametrize("enabled", [True, False])
@pytest.mark.parametrize("fails", [False, True])
def test_no_collection_during_a_capture(enabled, fails, monkeypatch):
    seen = []

    @contextlib.contextmanager
    def fake(g, **kw):
        seen.append((g, kw, gc.isenabled()))
        yield

    monkeypatch.setattr(torch.cuda, "graph", fake)
    was = gc.isenabled()
    (gc.enable if enabled else gc.disable)()
    try:
        with pytest.raises(ValueError) if fails else contextlib.nullcontext():
            with graph._capture("graph", pool="pool"):
                assert not gc.isenabled()
                if fails:
                    raise ValueError
        assert gc.isenabled() == enabled
    finally:
        (gc.enable if was else gc.disable)()
    assert seen == [("graph", {"pool": "pool"}, False)]


def test_a_dead_cycle_is_collected_before_the_capture_and_not_in_it(monkeypatch):
    gone = []

    class Held:
        def __init__(self, name):
            self.me, self.name = self, name          # a cycle: only the collector frees it

        def __del__(self):
            gone.append(self.name)

    monkeypatch.setattr(torch.cuda, "graph", lambda g, **kw: contextlib.nullcontext())
    Held("before")
    with graph._capture(None):
        assert gone == ["before"]
        Held("during")
        held = [[] for _ in range(30000)]            # objects enough to set the collector off
        assert gone == ["before"] and len(held) == 30000
    gc.collect()
    assert gone == ["before", "during"]
