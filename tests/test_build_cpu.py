"""When the build compiles again: a newer source, other flags, objects that nobody knows the flags of."""
import os
import stat

import pytest

from pyspark_tf_gke_amd._native import build as B

HIPCC = """#!/bin/sh
# writes what it is called with to the file behind -o
echo "$@" >> {log}
while [ $# -gt 1 ]; do [ "$1" = -o ] && out=$2; shift; done
for f in {root}/build/*.o; do [ "$f" = {root}/build/build_key.o ] && cat "$f"; done > "$out" 2>/dev/null
exit 0
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    (tmp_path / "csrc" / "kernels").mkdir(parents=True)
    for n in ("a", "b"):
        (tmp_path / "csrc" / "kernels" / f"{n}.hip").write_text("")
    cc = tmp_path / "hipcc"
    cc.write_text(HIPCC.format(log=tmp_path / "log", root=tmp_path))
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(cc))
    for k, v in (("CSRC", tmp_path / "csrc"), ("BUILD", tmp_path / "build"), ("HIP_LIB", tmp_path / "lib.so")):
        monkeypatch.setattr(B, k, v)

    def run(**kw):
        (tmp_path / "log").write_text("")
        B.build_hip(verbose=False, **kw)
        lines = (tmp_path / "log").read_text().splitlines()
        return sorted(os.path.basename(l.split(" -c ")[1].split()[0]) for l in lines if " -c " in l), \
            sum("-shared" in l for l in lines)

    run.root = tmp_path
    return run


def test_same_flags_build_once(tree):
    assert tree() == (["a.hip", "b.hip"], 1)
    assert tree() == ([], 0)
    for o in (tree.root / "build").glob("*.o"):  # a snapshot ships the library alone
        o.unlink()
    assert tree() == ([], 0)


def test_other_flags_compile_everything(tree):
    tree()
    assert tree(defines=("X=1",)) == (["a.hip", "b.hip"], 1)
    assert tree(defines=("X=1",)) == ([], 0)
    assert tree() == (["a.hip", "b.hip"], 1)


def test_objects_and_libraries_without_a_key_compile_again(tree):
    tree()
    (tree.root / "build" / "build_key").unlink()
    (tree.root / "lib.so").write_bytes(b"a library of unknown flags")
    assert tree() == (["a.hip", "b.hip"], 1)


def test_newer_source_compiles_alone(tree):
    tree()
    lib = (tree.root / "lib.so").stat().st_mtime
    os.utime(tree.root / "csrc" / "kernels" / "b.hip", (lib + 5, lib + 5))
    assert tree() == (["b.hip"], 1)


def test_flags_leave_out_packed_fp32_arithmetic(tree):
    tree()
    lines = [l for l in (tree.root / "log").read_text().splitlines() if " -c " in l]
    assert lines and all("-target-feature -Xclang -packed-fp32-ops" in l for l in lines)
