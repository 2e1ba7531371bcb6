"""Host logic of bench.py that needs no GPU: the config-5 bin packing."""
import importlib.util
import os

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _bench():
    spec = importlib.util.spec_from_file_location("bench", os.path.join(ROOT, "bench.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_pack_sequences_balanced_and_complete():
    b = _bench()
    for world in (1, 2, 4, 8):
        rng = np.random.default_rng(2)
        plen = np.exp(rng.uniform(np.log(128), np.log(8192), 64 * world)).astype(np.int64)
        members = b.pack_sequences(plen, world, 64)
        assert all(len(m) == 64 for m in members)
        flat = sorted(i for m in members for i in m)
        assert flat == list(range(64 * world))          # every sequence exactly once
        loads = [int(plen[m].sum()) for m in members]
        assert max(loads) - min(loads) <= int(plen.max())  # within one prompt of each other
    # one replica keeps the draw order
    rng = np.random.default_rng(2)
    plen = np.exp(rng.uniform(np.log(128), np.log(8192), 64)).astype(np.int64)
    assert b.pack_sequences(plen, 1, 64) == [list(range(64))]


def test_no_reference_library(monkeypatch, capsys):
    """A machine without the reference's library: its arm says so in its one line, and the
    library's own line keeps its figures and names the reason in cpu_baseline."""
    import json
    import types

    import oracle

    bench = _bench()

    def missing(self, variant=None):
        raise FileNotFoundError("libg4ref.so missing")
    monkeypatch.setattr(oracle.Reference, "__init__", missing)
    monkeypatch.setattr(oracle.Reference, "use_all_cores", staticmethod(lambda: None))
    bench.run_reference_arm(types.SimpleNamespace(gpus=1, steps=2, warmup=3), types.SimpleNamespace(rank=0, world=1))
    lines = capsys.readouterr().out.splitlines()
    assert [json.loads(x) for x in lines] == [{"impl": "reference", "unavailable": "libg4ref.so missing"}]
    assert bench.cpu_baseline(None) == {"unavailable": "libg4ref.so missing"}
