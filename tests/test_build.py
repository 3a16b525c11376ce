"""The library is built without torch, and its torch binding anew for another
torch (no GPU needed; both are up to date where these tests run)."""

import os
import subprocess
import sys

from opendressi_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_library_needs_no_torch():
    """Also where the binding is missing."""
    code = """
import sys
sys.modules["torch"] = None  # as if it were not installed
from opendressi_b200 import build
build.build()
build.BINDING = build.BINDING + ".missing"
assert build.build() == build.LIB
assert build.build(binding=False) == build.LIB
from opendressi_b200 import load_library
load_library()
"""
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, text=True,
                         capture_output=True, timeout=600)
    assert out.returncode == 0, out.stderr
    assert "binding of the learning operators is left out" in out.stderr


def test_another_torch_makes_the_binding_stale(monkeypatch):
    build.build()
    assert not build._binding_stale()
    monkeypatch.setattr(build, "_torch_version", lambda: "1.0")
    assert build._binding_stale()
