"""The calls on a paged cache: refusals and index arithmetic, checked without a GPU, and the layouts of their structs."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from cera_amd import hip_api as A

ROOT = Path(__file__).resolve().parent.parent
HEADER = (ROOT / "include" / "cera_hip.h").read_text()
SYS = (ROOT / "integration" / "cera-hip-sys" / "src" / "lib.rs").read_text()


def test_refusals_and_rows(tmp_path):
    exe = tmp_path / "paged_checks"
    b = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", f"-I{ROOT / 'cera_amd' / 'csrc'}", f"-I{ROOT / 'include'}",
                        str(ROOT / "tests" / "native" / "paged_checks.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert b.returncode == 0, b.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("name,cls,size", [("cera_hip_paged_kv", A.PagedKV, 72), ("cera_hip_paged_attn", A.PagedAttn, 112),
                                           ("cera_hip_paged_evict", A.PagedEvict, 48), ("cera_hip_verify_draft", A.VerifyDraft, 80)])
def test_structs_agree(name, cls, size):
    src = re.sub(r"/\*.*?\*/", "", HEADER, flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", src).group(1)
    fields = [re.sub(r"[\s\*]", "", part.split()[-1]) for decl in body.split(";") if decl.strip() for part in decl.split(",")]
    assert fields == [f[0] for f in cls._fields_]
    assert fields == re.findall(r"pub (\w+):", re.search(r"pub struct " + name + r" \{(.*?)\n\}", SYS, re.S).group(1))
    assert ctypes.sizeof(cls) == size and f"size_of::<{name}>(), {size}" in SYS


def test_a_null_context_is_refused():
    lib = A.load_library()
    assert lib.cera_hip_paged_attn_dev(None, A.PagedKV(), A.PagedAttn()) == 6
    assert lib.cera_hip_paged_evict_dev(None, A.PagedKV(), A.PagedEvict()) == 6
    assert lib.cera_hip_verify_draft_dev(None, A.VerifyDraft()) == 6
