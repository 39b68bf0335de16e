"""An incremental build recompiles what was compiled with other flags, and nothing else (a stand-in compiler writes its outputs down)."""
import os
import time

import pytest

FAKE = """#!/bin/sh
echo "$@" >> "$(dirname "$0")/log"
while [ $# -gt 0 ]; do if [ "$1" = -o ]; then shift; : > "$1"; fi; shift; done
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    from alphazero_amd import _build

    (tmp_path / "hipcc").write_text(FAKE)
    os.chmod(tmp_path / "hipcc", 0o755)
    srcs = [tmp_path / "a.hip", tmp_path / "b.hip"]
    for f in (*srcs, tmp_path / "h.hip.h", tmp_path / "_build.py"):
        f.write_text("x")
    monkeypatch.setenv("HIPCC", str(tmp_path / "hipcc"))
    monkeypatch.setattr(_build, "SRCS", [str(f) for f in srcs])
    monkeypatch.setattr(_build, "DEPS", [*[str(f) for f in srcs], str(tmp_path / "h.hip.h")])
    monkeypatch.setattr(_build, "RECIPE", str(tmp_path / "_build.py"), raising=False)
    monkeypatch.setattr(_build, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(_build, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(_build, "LIB", str(tmp_path / "lib.so"))

    def compiled():
        """the sources compiled by a build"""
        log = tmp_path / "log"
        log.unlink(missing_ok=True)
        _build.build()
        lines = log.read_text().splitlines() if log.exists() else []
        return sorted(os.path.basename(line.split()[-1]) for line in lines if " -c " in line), any("-shared" in line for line in lines)

    def later(name):
        """what was built becomes older than this file, and all else older still"""
        now = time.time()
        for f in tmp_path.rglob("*"):
            if f.is_file():
                os.utime(f, (now - 10,) * 2 if f.suffix in (".o", ".so") else (now - 20,) * 2)
        os.utime(tmp_path / name, (now - 5,) * 2)

    return _build, monkeypatch, compiled, later


def test_other_flags_recompile_everything(tree):
    build, monkeypatch, compiled, later = tree
    assert compiled() == (["a.hip", "b.hip"], True)
    assert compiled() == ([], False)
    monkeypatch.setattr(build, "FLAGS", [*build.FLAGS, "-DOTHER"])
    later("_build.py")  # (that is where the flags stand)
    assert compiled() == (["a.hip", "b.hip"], True)


def test_the_same_flags_recompile_what_is_newer(tree):
    build, monkeypatch, compiled, later = tree
    compiled()
    later("a.hip")
    assert compiled() == (["a.hip"], True)
    later("_build.py")
    assert compiled()[0] == []
