"""A library that lacks one of the calls is refused each time it is asked for, never handed out with calls whose types are not set."""
import subprocess

import pytest


def test_library_of_other_sources_is_refused_every_time(T, tmp_path, monkeypatch):
    from thrml_rs_b200 import _ffi
    (tmp_path / "old.c").write_text("int thrml_nothing(void) { return 0; }")
    old = tmp_path / "old.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(old), str(tmp_path / "old.c")], check=True)
    monkeypatch.setattr(_ffi, "_lib", None)
    monkeypatch.setattr(_ffi._build, "OUT", str(old))
    for _ in range(2):
        with pytest.raises(ImportError, match="other sources"):
            _ffi.lib()
