"""The library is built with hipcc alone; the module of the float operators' calls is beside it
where torch, a C++ compiler and Python's headers are.  (Stand-ins for the compilers.)"""
import os
import sys

import pytest

COMPILER = "#!/bin/sh\nwhile [ $# -gt 0 ]; do if [ \"$1\" = -o ]; then echo built > \"$2\"; fi; shift; done\n"


@pytest.fixture
def lib(tmp_path, monkeypatch):
    from mamba_int import build_lib
    cc = tmp_path / "cc"
    cc.write_text(COMPILER)
    cc.chmod(0o755)
    monkeypatch.setattr(build_lib, "HIPCC", str(cc))
    monkeypatch.setattr(build_lib, "CXX", str(cc))
    monkeypatch.setattr(build_lib, "LIB_PATH", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build_lib, "CALLS_PATH", str(tmp_path / "calls.so"))
    (tmp_path / "calls.so").write_text("of another build")
    return build_lib


def test_both_are_built(lib):
    assert lib.build() == lib.LIB_PATH and os.path.exists(lib.LIB_PATH)
    assert open(lib.CALLS_PATH).read() == "built\n"


@pytest.mark.parametrize("missing", ["compiler", "torch", "headers"])
def test_the_library_alone(lib, missing, monkeypatch, tmp_path, capsys):
    if missing == "compiler":
        monkeypatch.setattr(lib, "CXX", str(tmp_path / "none"))
    elif missing == "torch":
        import importlib.util
        find = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
        monkeypatch.setitem(sys.modules, "torch", None)
    else:
        paths = lib.sysconfig.get_paths()
        monkeypatch.setattr(lib.sysconfig, "get_paths", lambda: {**paths, "include": str(tmp_path)})
    assert lib.build() == lib.LIB_PATH and os.path.exists(lib.LIB_PATH)
    assert not os.path.exists(lib.CALLS_PATH)
    assert "left out" in capsys.readouterr().err


def test_an_error_of_the_module_leaves_the_library(lib, monkeypatch, tmp_path):
    bad = tmp_path / "bad"
    bad.write_text("#!/bin/sh\necho no such thing >&2\nexit 3\n")
    bad.chmod(0o755)
    monkeypatch.setattr(lib, "CXX", str(bad))
    with pytest.raises(RuntimeError, match="no such thing"):
        lib.build()
    assert os.path.exists(lib.LIB_PATH) and not os.path.exists(lib.CALLS_PATH)
