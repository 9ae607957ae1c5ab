"""What the host allows and refuses of the calls on a paged cache, checked without a GPU."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_allowed_and_refused(tmp_path):
    exe = tmp_path / "paged_contract"
    b = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", f"-I{ROOT / 'cera_amd' / 'csrc'}", f"-I{ROOT / 'include'}",
                        str(ROOT / "tests" / "native" / "paged_contract.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert b.returncode == 0, b.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
