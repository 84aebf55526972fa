"""The build entry point where torch cannot be imported: the CKKS package needs none."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

CODE = """
import importlib.util, sys, types
sys.modules["torch"] = None  # `import torch` raises ImportError
sys.path.insert(0, {root!r})
import __graft_entry__ as entry
real = importlib.util.spec_from_file_location
importlib.util.spec_from_file_location = lambda name, path: real(name, {stub!r})
sys.modules["oracle"] = types.SimpleNamespace(build=lambda: "oracle")
entry.build()
assert "easyfhe" in sys.modules and "clear_model" not in sys.modules
"""


def test_build_without_torch(tmp_path):
    """Everything but the compilations, which are the same either way."""
    stub = tmp_path / "build.py"
    stub.write_text("CLEAR_LIB = 'clear'\ndef build():\n    return 'ckks'\n")
    code = CODE.format(root=str(ROOT), stub=str(stub))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert "clear_model" in r.stdout  # says what it left out
