"""The default make target on machines with and without PyTorch: the C library needs none."""
import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "xiaomi-hexagon-exl3_amd"


def plan(*args):
    """the commands of make, none of them run"""
    return subprocess.run(["make", "-n", "-B", *args], cwd=PKG, capture_output=True, text=True, timeout=120)


@pytest.fixture
def no_torch(tmp_path):
    exe = tmp_path / "python"
    exe.write_text(f"#!/bin/sh\nexec {sys.executable} -I -S \"$@\"\n")  # without site-packages
    exe.chmod(0o755)
    return f"PYTHON={exe}"


def test_default_target_without_torch(no_torch):
    r = plan("all", no_torch)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "-o libexl3_hip.so" in r.stdout and "-o libexl3_hip_stamps.so" in r.stdout
    assert "exl3_torch.cpp" not in r.stdout
    assert "exl3_torch.so" in r.stdout  # says what was left out


def test_torch_module_asked_for_without_torch(no_torch):
    r = plan("exl3_torch.so", no_torch)
    assert r.returncode != 0 and "PyTorch" in r.stderr


def test_default_target_with_torch():
    r = plan("all", f"PYTHON={sys.executable}")
    assert r.returncode == 0, r.stderr[-2000:]
    assert "-o exl3_torch.so" in r.stdout
