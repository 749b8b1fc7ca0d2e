"""What the build needs."""
import sys

from visualmesh_b200 import build


def test_the_engine_is_built_without_torch(monkeypatch, capsys):
    built = []
    monkeypatch.setattr(build, "_module_stale", lambda module: True)
    monkeypatch.setattr(build, "_library_stale", lambda: False)
    monkeypatch.setattr(build, "_build_module", lambda module, more: built.append(module))
    for name in ["torch"] + [m for m in sys.modules if m.startswith("torch.")]:
        monkeypatch.setitem(sys.modules, name, None)
    assert build.build() == build.LIB
    assert built == [build.NATIVE] and "torch" in capsys.readouterr().err
    monkeypatch.setattr(build, "_module_stale", lambda module: module == build.ANSWERS)
    assert not build.needs_build()
    monkeypatch.delitem(sys.modules, "torch")
    assert build.needs_build()
