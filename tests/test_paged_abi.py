"""CPU-side checks of include/sage_paged_b200.h: it stands alone in C and C++, and the library exports what it declares."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from sageattention_rdna3_b200 import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sage_paged_b200.h")


def declared_symbols():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(sage_[a-z0-9_]+)\s*\(", text)))


def test_library_exports_what_the_header_declares():
    assert declared_symbols() == ["sage_apply_rotary", "sage_paged_append", "sage_paged_attn", "sage_paged_workspace_bytes"]
    lib = ctypes.CDLL(str(_native.ABI_PATH))
    for name in declared_symbols():
        assert hasattr(lib, name), f"{name} is declared but not exported"


@pytest.mark.parametrize("compiler, language", [("gcc", "c"), ("g++", "c++")])
def test_header_stands_alone(compiler, language):
    if shutil.which(compiler) is None:
        pytest.skip(f"{compiler} is not installed")
    subprocess.run([compiler, "-x", language, "-Wall", "-Werror", "-fsyntax-only", HEADER], check=True)


def test_operators_are_registered():
    ops = _native.load_ops()
    for name in ("rotary", "paged_append", "paged_attn"):
        getattr(ops, name)
