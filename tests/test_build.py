"""The library's build where the Python binding cannot be built."""
import os
import shutil
import subprocess
import sys

from ai_engine_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_without_torch(tmp_path):
    """A C caller's build: no torch (-S leaves installed packages out)."""
    build.build()
    for d in ("ai_engine_b200/csrc", "ai_engine_b200/_build", "include"):
        shutil.copytree(os.path.join(ROOT, d), tmp_path / d)
    script = shutil.copy2(os.path.join(ROOT, "ai_engine_b200", "build.py"), tmp_path / "ai_engine_b200")
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    assert subprocess.run([sys.executable, "-S", "-c", "import torch"], env=env, capture_output=True).returncode
    r = subprocess.run([sys.executable, "-S", script, "--changed"], env=env, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert (tmp_path / "ai_engine_b200" / "libaie_conv.so").exists()
    assert not (tmp_path / "ai_engine_b200" / "_seqcall.so").exists()
    assert "_seqcall.so is left out: torch not found" in r.stderr


def test_binding_without_python_headers(monkeypatch, tmp_path):
    assert build.bind_needs() == ""
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert build.bind_needs() == "Python's headers"
