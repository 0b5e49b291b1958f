"""A library that is not this package's is refused by what is wrong with it (no GPU needed)."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
LOAD = """
import importlib, sys
from pathlib import Path
qs = importlib.import_module("quant-studio_amd")
qs._lib, qs.LIB_PATH = None, Path(sys.argv[1])      # the package's own is loaded by its import
try:
    qs.library()
except ImportError as e:
    print("ImportError:", e)
"""


@pytest.mark.parametrize("version,word", [(3, "ABI version 3 != 4"), (5, "ABI version 5 != 4"), (4, "older build"),
                                          (None, "lacks qs_abi_version")])
def test_other_libraries(tmp_path, version, word):
    """Of another version, and of this one before functions were added to it."""
    source, lib = tmp_path / "lib.c", tmp_path / "libqs_hip.so"
    source.write_text("int other;\n" if version is None else f"int qs_abi_version(void) {{ return {version}; }}\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(source)], check=True)
    r = subprocess.run([sys.executable, "-c", LOAD, str(lib)], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.startswith("ImportError:") and word in r.stdout, r.stdout + r.stderr
