"""csrc/build.py: when a library is out of date."""
import os

import pytest

from custom_d_fine_amd.csrc import build


@pytest.mark.parametrize("newer", ["attn.hip", "common.h", "runtime.cpp", "dfine_hip.h", "build.py"])
def test_library_is_out_of_date(tmp_path, monkeypatch, newer):
    """A source, a header, the interface's header or the flags (build.py) changed after the library was built."""
    lib = tmp_path / "lib.so"
    lib.write_bytes(b"")
    monkeypatch.setattr(build, "LIB", str(lib))
    times = {}
    monkeypatch.setattr(build.os.path, "getmtime", lambda p: 2 if p == str(lib) else times.get(os.path.basename(p), 1))
    assert not build.needs_build()
    times[newer] = 3
    assert build.needs_build()


def test_the_build_entry_compiles_each_time(monkeypatch):
    import __graft_entry__ as entry
    asked = []
    monkeypatch.setattr(build, "build", lambda force=False, verbose=True: asked.append(force) or build.LIB)
    monkeypatch.setattr(entry.subprocess, "check_call", lambda *a, **k: 0)
    entry.build()
    assert asked == [True]
