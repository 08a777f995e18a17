"""The build's order of work (nothing is compiled here)."""
import os

import pytest

from sparc_amd import build as B


def test_the_library_is_linked_without_the_torch_binding(tmp_path, monkeypatch):
    """Callers of the C library need neither torch's headers nor g++."""
    def run(cmd, what):
        out = cmd[cmd.index("-o") + 1]
        assert out.startswith(str(tmp_path))
        with open(out, "w") as f:
            f.write(what)

    def no_binding(build_dir):
        raise RuntimeError("no headers")

    for name, file in (("HERE", ""), ("LIB_PATH", B.LIB_NAME), ("NATIVE_PATH", "_native.so")):
        monkeypatch.setattr(B, name, str(tmp_path / file))
    monkeypatch.setattr(B, "_run", run)
    monkeypatch.setattr(B, "_compile_native", no_binding)
    with pytest.raises(RuntimeError, match="no headers"):
        B.build()
    assert os.path.exists(B.LIB_PATH) and not os.path.exists(B.NATIVE_PATH)
