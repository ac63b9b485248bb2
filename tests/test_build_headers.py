"""A change of any header that a source includes rebuilds it."""
from __future__ import annotations

import importlib.util
import re
from pathlib import Path

REPO = Path(__file__).resolve().parents[1]
PKG = REPO / "orin-cuda-operator-library_b200"


def test_every_included_header_is_a_dependency():
    spec = importlib.util.spec_from_file_location("opl_build", PKG / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    known = set(build._headers())
    sources = [*(PKG / "csrc").iterdir(), *(PKG / "python").glob("*.cpp")]
    for source in (p for p in sources if p.suffix in (".cu", ".cuh", ".h", ".cpp")):
        for name in re.findall(r'#include "([^"]+)"', source.read_text()):
            found = [p for p in (PKG / "csrc" / name, REPO / "include" / name) if p.exists()]
            assert found and found[0] in known, (source.name, name)
