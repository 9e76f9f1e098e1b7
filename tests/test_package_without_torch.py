"""The package where torch, or the module over its tensors, is not there: everything but the operators over torch
tensors works."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCK = """
import sys
class Block:
    def find_spec(self, name, path=None, target=None):
        if name.split(".")[-1] == sys.argv[2]:
            raise ModuleNotFoundError("blocked", name=name)
sys.meta_path.insert(0, Block())
sys.path.insert(0, sys.argv[1])
"""


def run(code, blocked):
    return subprocess.run([sys.executable, "-c", BLOCK + code, ROOT, blocked], capture_output=True, text=True, timeout=300)


@pytest.mark.parametrize("blocked", ["torch", "_torch_call"])
def test_star_import(blocked):
    r = run("""
from crosslane_b200 import *
assert pack and ExpertBank and route_host
assert "ExpertRoute" not in globals()
import crosslane_b200
try:
    crosslane_b200.ExpertRoute
except ImportError as e:
    print("refused", e)
""", blocked)
    assert r.returncode == 0 and "refused" in r.stdout, r.stderr[-1500:]


def test_star_import_with_torch():
    pytest.importorskip("torch")
    r = run("""
from crosslane_b200 import *
assert ExpertRoute and BlockNorm and Int8Linear and int8_quantize and pack
""", "nothing")
    assert r.returncode == 0, r.stderr[-1500:]


def test_names_are_listed():
    import crosslane_b200
    assert {"ExpertRoute", "BlockNorm", "Int8Linear", "int8_quantize", "ExpertBank"} <= set(dir(crosslane_b200))
    with pytest.raises(AttributeError):
        crosslane_b200.no_such_name
