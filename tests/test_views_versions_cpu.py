"""The compiled argument packing is used with the torch and the Python that it was compiled for, and with no other."""
import subprocess
import sys

import pytest
import torch

from g4b_b200 import _cabi

FRESH = """
import sys
from g4b_b200 import _cabi
_cabi.load()
assert "torch" not in sys.modules and _cabi._fast is None
import torch
x = torch.zeros(2, 3)
first = _cabi.views(x)
assert _cabi._fast is not None
assert first == _cabi._fast.views(False, (x,))
"""


def test_torch_imported_behind_the_library():
    if subprocess.run([sys.executable, "-c", "import sys; from g4b_b200 import _cabi; _cabi.load(); sys.exit('torch' in sys.modules)"]).returncode:
        pytest.skip("torch comes with the interpreter here")
    code = FRESH.replace("first = ", "_cabi._validate_only_depth = 1\nfirst = ")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


@pytest.fixture
def anew(monkeypatch):
    _cabi.load()
    monkeypatch.setattr(_cabi, "_fast", None)
    monkeypatch.setattr(_cabi, "_fast_looked_for", False)


def test_this_torch_and_python(anew):
    _cabi._load_fast()
    assert _cabi._fast is not None and torch.__version__ in _cabi._fast.built_for


@pytest.mark.parametrize("other", ["torch", "python", "implementation"])
def test_another_torch_or_python(anew, monkeypatch, other):
    if other == "torch":
        monkeypatch.setattr(torch, "__version__", torch.__version__ + "x")
    elif other == "python":
        monkeypatch.setattr(sys, "version", "3.99.0 (another)")
    else:
        monkeypatch.setattr(sys.implementation, "cache_tag", "other-312")
    x = torch.zeros(2, 3)
    _cabi.views(x)
    assert _cabi._fast is None                      # and stays so: one look
    monkeypatch.undo()


def test_a_module_without_the_mark(anew, monkeypatch, tmp_path):
    """One that was built before it carried any."""
    import importlib.util

    real = importlib.util.module_from_spec
    spec_of = importlib.util.spec_from_file_location

    class Old:
        def create_module(self, spec):
            return None

        def exec_module(self, module):
            pass

    monkeypatch.setattr(importlib.util, "spec_from_file_location", lambda name, path: spec_of(name, path, loader=Old()))
    monkeypatch.setattr(importlib.util, "module_from_spec", real)
    _cabi._load_fast()
    assert _cabi._fast is None and _cabi._fast_looked_for
