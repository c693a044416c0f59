"""The hold that a call of several launches has on its stream's internal workspace (csrc/exl3_workspace.hpp), on the host
with ThreadSanitizer; and every call that takes an internal workspace keeps the hold until it returns."""
import re
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "xiaomi-hexagon-exl3_amd" / "csrc"


def test_launches_of_a_call_keep_together(tmp_path):
    exe = tmp_path / "workspace_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=thread", "-Wall", "-Wextra", f"-I{CSRC}", "-o", str(exe),
                    str(ROOT / "tests" / "cpp" / "workspace_check.cpp"), "-pthread"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr[-3000:]


def test_every_taker_declares_its_lease():
    """a lease that dies before the last launch would hold nothing: it is declared in the entry itself, outside any block
    that ends before the launches"""
    for name in ("exl3_api.cpp", "exl3_attention_api.cpp"):
        text = (CSRC / name).read_text()
        bodies = {m.group(1): m.group(0) for m in re.finditer(
            r"^(?:static )?exl3_status (exl3_hip_\w+|mul_mat_impl)\(.*?^}", text, re.S | re.M)}
        takers = [n for n, b in bodies.items() if re.search(r"\b(call_workspace|take_workspace)\(", b)]
        assert takers
        for n in takers:
            assert re.search(r"^    exl3k::WorkspaceLease lease;$", bodies[n], re.M), n
