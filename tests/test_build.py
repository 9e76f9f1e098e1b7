"""build.py: the CUDA library is built whatever torch is installed, and the module over torch tensors for the torch and
the Python that are."""
import importlib.util
import os
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def b(tmp_path, monkeypatch):
    """build.py with its outputs under tmp_path, compilers that only write their output, and a made-up torch."""
    spec = importlib.util.spec_from_file_location("clb_build_test", os.path.join(ROOT, "crosslane_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    monkeypatch.setattr(b, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(b, "TORCH_CALL", str(tmp_path / os.path.basename(b.TORCH_CALL)))
    b.ran, b.fails = [], set()

    def run(cmd, **kw):
        b.ran.append(cmd[0])
        if cmd[0] in b.fails:
            return types.SimpleNamespace(returncode=1, stdout="", stderr="no")
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("x")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    def torch(name, cuda=True, version="1"):
        home = tmp_path / name
        (home / "lib").mkdir(parents=True, exist_ok=True)
        (home / "version.py").write_text(f"__version__ = {version!r}")
        os.utime(home / "version.py", (1, 1))  # an old file, as in a package of some time ago
        if cuda:
            (home / "lib" / "libc10_cuda.so").write_text("")
        b.origin = str(home / "__init__.py")

    monkeypatch.setattr(b.subprocess, "run", run)
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: types.SimpleNamespace(origin=b.origin) if b.origin else None)
    b.torch, b.origin = torch, None
    return b


def test_without_torch_or_with_one_without_cuda(b):
    b.build()
    assert os.path.exists(b.LIB) and b.CXX not in b.ran
    b.torch("cpu_only", cuda=False)
    b.build()
    assert b.CXX not in b.ran and not os.path.exists(b.TORCH_CALL)


def test_the_library_is_linked_before_the_module_fails(b):
    b.torch("torch")
    b.fails.add(b.CXX)
    with pytest.raises(RuntimeError, match="torch_call.cpp"):
        b.build()
    assert os.path.exists(b.LIB)


def test_the_module_is_built_for_the_torch_that_is_there(b):
    b.torch("one")
    b.build()
    b.build()
    assert b.ran.count(b.CXX) == 1
    b.torch("one", version="2")  # replaced in place
    b.build()
    b.torch("two", version="2")  # another environment
    b.build()
    b.build()
    assert b.ran.count(b.CXX) == 3
    b.build(force=True)
    assert b.ran.count(b.CXX) == 4


def test_the_module_is_named_for_this_python(b):
    import sysconfig
    assert b.TORCH_CALL.endswith("_torch_call" + sysconfig.get_config_var("EXT_SUFFIX"))
