"""CPU: what counts as out of date, and the library without its binding."""

import pytest
import torch

from preemptlm_b200 import build


def test_another_torch_makes_the_binding_stale(monkeypatch):
    build.build_library()
    assert not build.is_stale()
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "0.0.1")
        assert build.is_stale()
    assert not build.is_stale()


def test_library_without_binding(monkeypatch, tmp_path):
    """The library is built and stays where it is when the binding does not compile."""
    (tmp_path / "a.cu").write_text("extern \"C\" int sg_nothing() { return 0; }\n")
    monkeypatch.setattr(build, "sources", lambda: [tmp_path / "a.cu"])
    for name, path in (("BUILD_DIR", "_build"), ("LIB_DIR", "lib"), ("LIB_PATH", "lib/libsg_b200.so"),
                       ("BINDING_PATH", "_native.so"), ("BINDING_SRC", "binding.cpp"), ("BINDING_STAMP", "_build/binding.txt")):
        monkeypatch.setattr(build, name, tmp_path / path, raising=False)
    (tmp_path / "binding.cpp").write_text("#error no such torch\n")
    (tmp_path / "_native.so").write_text("of another torch")
    with pytest.warns(RuntimeWarning, match="no such torch"):
        path = build.build_library()
    assert path.exists() and not (tmp_path / "_native.so").exists()
    built = path.stat().st_mtime_ns
    with pytest.warns(RuntimeWarning, match="no such torch"):  # said every time, and the library is not built again
        build.build_library()
    assert path.stat().st_mtime_ns == built
