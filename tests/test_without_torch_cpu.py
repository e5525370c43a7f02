"""The package on a Python that has no torch: everything but the operators on torch tensors."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _python(code, torch):
    block = "" if torch else "import sys; sys.modules['torch'] = None\n"
    r = subprocess.run([sys.executable, "-c", block + code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return r.stdout.split()


@pytest.mark.parametrize("torch", [False, True])
def test_star_import(torch):
    assert _python("from symplex_b200 import *\nprint(callable(gemm_host), 'layer_norm' in dir(), 'int4_matvec' in dir())", torch) == \
        ["True", str(torch), str(torch)]


@pytest.mark.parametrize("torch", [False, True])
def test_hasattr_answers(torch):
    assert _python("import symplex_b200 as sx\nprint(hasattr(sx, 'layer_norm'), hasattr(sx, 'gemm'), hasattr(sx, 'no_such_name'))", torch) == \
        [str(torch), "True", "False"]


def test_the_reason_is_named():
    code = "import symplex_b200 as sx\ntry:\n    sx.int4_quantize\nexcept AttributeError as e:\n    print('torch' in str(e), type(e.__cause__).__name__)"
    assert _python(code, False) == ["True", "ModuleNotFoundError"]


def test_importing_the_package_does_not_import_torch():
    assert _python("import sys, symplex_b200\nprint('torch' in sys.modules)", True) == ["False"]
