"""What the package Makefile builds where torch is there and where it is not
(dry runs)."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "bnn-train-infer_b200"


def commands(*args):
    """What make would run if every source had changed."""
    got = subprocess.run(["make", "-n", "-B", "-C", str(PKG), *args], capture_output=True, text=True, timeout=120)
    assert got.returncode == 0, got.stderr
    return got.stdout


def script(path, text):
    path.write_text("#!/bin/sh\n" + text)
    path.chmod(0o755)
    return f"PYTHON={path}"


@pytest.mark.parametrize("text", ["exit 127", f'exec {sys.executable} -S -E "$@"'])  # no Python; a Python without torch
def test_library_and_cli_need_no_torch(tmp_path, text):
    got = commands(script(tmp_path / "python", text))
    assert "libbnn_b200.so" in got and "bnn-infer-b200" in got
    assert "paged_torch.cpp" not in got


def test_binding_is_built_beside_torch(tmp_path):
    pytest.importorskip("torch")
    assert "paged_torch.cpp" in commands(f"PYTHON={sys.executable}")


def test_binding_follows_torch(tmp_path):
    """Another torch under the same Python: the binding is built again, else not."""
    pytest.importorskip("torch")
    log, stamp, made = tmp_path / "log", tmp_path / "torch", tmp_path / "binding.so"
    tools = tmp_path / "tools"
    tools.mkdir()
    script(tools / "g++", f"echo called >> {log}\ntouch {made}\n")

    def builds():
        subprocess.run(["make", "-C", str(PKG), str(made), f"BUILD={tmp_path}", f"BINDING={made}", f"PYTHON={sys.executable}"], check=True,
                       capture_output=True, timeout=120, env={**os.environ, "PATH": f"{tools}:{os.environ['PATH']}"})
        return log.read_text().count("called")

    assert builds() == 1
    assert builds() == 1
    stamp.write_text("another torch\n")
    os.utime(made, (stamp.stat().st_mtime - 10,) * 2)
    assert builds() == 2


@pytest.mark.parametrize("checkout", [False, True])
def test_checkers_are_built_where_the_reference_is(tmp_path, monkeypatch, checkout):
    """An empty folder in its place is no reason to fail."""
    import __graft_entry__ as entry
    if checkout:
        (tmp_path / "bnn-accelerator").mkdir()
    ran = []
    monkeypatch.setattr(entry, "REFERENCE", tmp_path)
    monkeypatch.setattr(entry.subprocess, "run", lambda command, **kw: ran.append(command))
    entry.build()
    assert any("ref" in command for command in ran) == checkout
