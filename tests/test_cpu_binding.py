"""The native torch binding: what works without it, and when it is built."""
import subprocess
import sys
from pathlib import Path

import pytest

pytest.importorskip("torch")

REPO = Path(__file__).resolve().parent.parent


def test_ops_without_the_binding():
    """A tree whose _bind.so does not fit the installed torch: every operator of
    the ctypes binding is there, the four that need it say so when called."""
    code = """
import sys
sys.modules["pixal3d.cpp_b200._bind"] = None
from pixal3d.cpp_b200 import flow, ops
import torch
assert callable(ops.linear) and callable(ops.varlen_attention)
x = torch.zeros((2, 16))
for call in (lambda: ops.quantize_rows(x), lambda: ops.rotary(x, x[0].double(), 1, 16),
             lambda: ops.linear_i8(x, x, x, x), lambda: ops.masked_attention(x, x, x, x, x, 1, 1, 1, 1.0)):
    try:
        call()
    except ImportError as e:
        assert "_bind.so" in str(e)
    else:
        raise SystemExit("not refused")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.fixture
def builds(monkeypatch, tmp_path):
    """_build_bind with its compiler call replaced by one that makes the file."""
    from pixal3d.cpp_b200 import build as b
    ran = []

    def run(cmd, verbose):
        ran.append(cmd)
        b.BIND_LIB.write_text("")

    monkeypatch.setattr(b, "BIND_LIB", tmp_path / "_bind.so")
    if hasattr(b, "BIND_STAMP"):
        monkeypatch.setattr(b, "BIND_STAMP", tmp_path / "stamp")
    monkeypatch.setattr(b, "_run", run)
    return b, ran


def _torch_at(monkeypatch, where):
    import importlib.util
    import types
    spec = None if where is None else types.SimpleNamespace(origin=str(where / "__init__.py"))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec)


def test_build_without_torch(builds, monkeypatch, capsys):
    """The C and C++ libraries need no torch, so neither does building them."""
    b, ran = builds
    _torch_at(monkeypatch, None)
    b._build_bind(False, False)
    assert not ran and "torch" in capsys.readouterr().err


def test_binding_is_rebuilt_for_another_torch(builds, monkeypatch, tmp_path):
    """Whatever the times of its files are."""
    import os
    b, ran = builds
    for i, version in enumerate(("2.0", "2.1")):
        d = tmp_path / f"torch{i}"
        d.mkdir()
        (d / "version.py").write_text(f"__version__ = '{version}'")
        os.utime(d / "version.py", (1000.0, 1000.0))
        _torch_at(monkeypatch, d)
        b._build_bind(False, False)
        assert len(ran) == i + 1
        b._build_bind(False, False)
        assert len(ran) == i + 1
    (tmp_path / "torch1" / "version.py").write_text("__version__ = '2.1.1'")
    os.utime(tmp_path / "torch1" / "version.py", (1000.0, 1000.0))
    b._build_bind(False, False)
    assert len(ran) == 3
