"""The generation that tells whether a captured graph still holds a live address moves whenever the address goes, also when the
new allocation then fails: nvk_hip_util.h over an allocator that fails when told to (tests/workspace_driver.cpp), no device."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "nano_vllm_amd", "csrc")


def test_growth_with_an_allocator_that_fails(tmp_path):
    rocm = "/opt/rocm/include"
    if shutil.which("g++") is None or not os.path.isdir(rocm):
        pytest.skip("no host compiler or HIP headers")
    exe = str(tmp_path / "workspace_driver")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-D__HIP_PLATFORM_AMD__", "-I", rocm, "-I", os.path.join(ROOT, "include"), "-I", CSRC,
                        "-o", exe, os.path.join(ROOT, "tests", "workspace_driver.cpp"), "-lpthread"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_buffers_with_a_generation_grow_through_the_checked_helpers():
    """(so that the test above speaks for all of them: the split-K workspace, the decode plan, the 4-bit pool, the block index)"""
    for name, least in (("nvk_paged_attn.hip", 5), ("nvk_mx4.hip", 2), ("nvk_sparse.hip", 2)):
        text = open(os.path.join(CSRC, name)).read()
        assert len(re.findall(r"nvk::grow_(?:buffer|counters)\(", text)) >= least, name
        assert not re.search(r"generation\s*\+\+|\+\+\s*\w+->\w*generation", text), f"{name}: a generation is counted outside the helpers"
    batch = open(os.path.join(CSRC, "nvk_batch.hip")).read()
    body = batch[batch.index("int reserve_hidden_rows("):]
    assert body.index("hidden_generation++") < body.index("hipFree("), "the scratch rows' generation moves before they are freed"
