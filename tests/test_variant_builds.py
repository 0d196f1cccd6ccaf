"""tools/build_variants.sh and `make asm` build the sources of the shipped library with its flags (run over a compiler that only writes
down how it was called)."""
import glob
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COMPILER = """#!/bin/bash
echo "$@" >> "$CALLS"
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then mkdir -p "$(dirname "$2")" && : > "$2"; fi
  shift
done
"""


@pytest.fixture
def tree(tmp_path):
    if shutil.which("make") is None:
        pytest.skip("no make")
    for part in ("Makefile", "tools/build_variants.sh", "tools/nvk_run.cpp"):
        os.makedirs(os.path.dirname(tmp_path / part), exist_ok=True)
        shutil.copy(os.path.join(ROOT, part), tmp_path / part)
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    shutil.copytree(os.path.join(ROOT, "nano_vllm_amd", "csrc"), tmp_path / "nano_vllm_amd" / "csrc")
    cc = tmp_path / "hipcc"
    cc.write_text(COMPILER)
    cc.chmod(0o755)
    return tmp_path


def run(tree, *cmd):
    log = tree / "calls"
    log.write_text("")
    env = dict(os.environ, HIPCC=str(tree / "hipcc"), CALLS=str(log))
    env.pop("MAKEFLAGS", None)
    r = subprocess.run(cmd, cwd=tree, env=env, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    return [line.split() for line in log.read_text().splitlines()]


def compiled(calls):
    """source -> the flags it was compiled with, names of files aside"""
    out = {}
    for c in calls:
        for w in c:
            if w.endswith((".hip", ".cpp")):
                out[os.path.basename(w)] = [x for x in c if "/" not in x and x not in ("-o", "-c")]
    return out


def test_variants_are_the_library_with_more_flags(tree):
    shipped = run(tree, "make", "lib")
    variant = run(tree, "bash", "tools/build_variants.sh", "one:-DNVK_X=1 -DNVK_Y=2", "plain")
    lib, var = compiled(shipped), compiled(variant)
    assert sorted(lib) == sorted(os.path.basename(p) for p in glob.glob(os.path.join(ROOT, "nano_vllm_amd", "csrc", "*.[hc][ip]p")))
    assert (tree / "build/variants/one.so").exists() and (tree / "build/variants/plain.so").exists()
    for out, more in (("one", ["-DNVK_X=1", "-DNVK_Y=2"]), ("plain", [])):
        mine = [c for c in variant if any(f"/obj_{out}/" in w or w.endswith(f"/{out}.so") for w in c)]
        got = compiled(mine)
        assert sorted(got) == sorted(lib)
        for name, flags in got.items():
            assert flags == lib[name] + (more if name.endswith(".hip") else []), name
        link = [c for c in mine if "-shared" in c]
        assert len(link) == 1 and sum(w.endswith(".o") for w in link[0]) == len(lib)


def test_the_register_report_is_of_the_shipped_kernels(tree):
    lib, asm = compiled(run(tree, "make", "lib")), compiled(run(tree, "make", "asm"))
    assert sorted(asm) == sorted(n for n in lib if n.endswith(".hip"))
    for name, flags in asm.items():
        assert [f for f in flags if f not in ("-save-temps=obj", "-Rpass-analysis=kernel-resource-usage")] == lib[name], name
