"""What is built, and from what: the library without torch, the binding by the torch
it was built against."""
import subprocess
import sys
import sysconfig
from pathlib import Path

import pytest
import torch

from fp4_sm120a_b200 import _native, build


def test_library_without_torch(nvlib, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.binding_path() is None
    assert not build.needs_build()
    assert build.build() == build.LIB
    monkeypatch.setattr(build, "_run", lambda *a: None)      # as if the library were old
    monkeypatch.setattr(build, "needs_build", lambda: True)
    assert build.build() == build.LIB
    assert "no torch" in capsys.readouterr().err


def test_build_script_imports_no_package():
    """As a C or C++ user calls it: torch is not looked for before nvcc is done."""
    code = ("import sys, runpy; sys.modules['torch'] = None; "
            "m = runpy.run_path(sys.argv[1]); assert m['binding_path']() is None")
    script = Path(build.__file__)
    subprocess.run([sys.executable, "-c", code, str(script)], check=True, timeout=120)


@pytest.mark.parametrize("compiler", ["/bin/false", "/nonexistent/g++"])
def test_library_without_a_host_compiler(nvlib, monkeypatch, capsys, tmp_path, compiler):
    """The binding fails by itself, and no old one is left to be imported."""
    old = tmp_path / "_torch_binding.so"
    old.write_bytes(b"of another version")
    monkeypatch.setattr(build, "binding_path", lambda: old)
    monkeypatch.setattr(build, "_binding_deps", lambda: [build.BINDING_SOURCE, build.LIB, old])
    monkeypatch.setattr(build, "_stale", lambda target, deps: target == old)
    monkeypatch.setattr(build, "CXX", compiler)
    assert build.build() == build.LIB
    assert not old.exists()
    assert "not built" in capsys.readouterr().err


def test_binding_is_named_by_python_and_torch(nvlib, monkeypatch):
    name = build.binding_path().name
    assert torch.__version__ in name and sysconfig.get_config_var("SOABI") in name
    assert _native.load_binding().__file__ == str(build.binding_path())
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    monkeypatch.setattr(_native, "_binding", None)
    with pytest.raises(ImportError, match="0.0.1"):
        _native.load_binding()
