"""Between a matrix instruction and the first other instruction that touches its result the compiler has to leave so many issue slots
(the hardware does not wait by itself).  A build was seen whose first read stood one slot behind, across a branch, and whose scores
differed from run to run; so every path of the shipped kernels is walked here.  How many slots an instruction takes is read
off a straight line of the same compiler's, which fills it up with s_nop to the slot."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "nano_vllm_amd", "libnvk_paged_attn.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
HIPCC = "/opt/rocm/bin/hipcc"
MOST = 24  # slots that a walk looks ahead

STRAIGHT = """
#include <hip/hip_runtime.h>
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16 __attribute__((ext_vector_type(16)));
typedef double d4 __attribute__((ext_vector_type(4)));
__global__ void one(f4 *o, const b8 *p) { f4 c = o[0]; c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p[0], p[1], c, 0, 0, 0); o[0] = c * 3.f; }
__global__ void two(d4 *o, const double *p) { d4 c = o[0]; c = __builtin_amdgcn_mfma_f64_16x16x4f64(p[0], p[1], c, 0, 0, 0); o[0] = c * 3.0; }
__global__ void three(f4 *o, const float *p) { f4 c = o[0]; c = __builtin_amdgcn_mfma_f32_16x16x4f32(p[0], p[1], c, 0, 0, 0); o[0] = c * 3.f; }
__global__ void four(f16 *o, const float *p) { f16 c = o[0]; c = __builtin_amdgcn_mfma_f32_32x32x2f32(p[0], p[1], c, 0, 0, 0); o[0] = c * 3.f; }
"""


def registers(token):
    m = re.match(r"^[-|]*([av])\[(\d+):(\d+)\]", token)
    if m:
        return {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.match(r"^[-|]*([av])(\d+)\b", token)
    return {(m[1], int(m[2]))} if m else set()


def functions(text):
    """name -> [(address, opcode, operands, branch target or None)] of a disassembly"""
    out, cur, start = {}, None, {}
    for line in text.splitlines():
        m = re.match(r"^([0-9a-f]{16}) <(.+)>:$", line)
        if m:
            cur = out[m[2]] = []
            start[m[2]] = int(m[1], 16)
            continue
        m = re.match(r"^\t(\S+)(.*?)//\s*([0-9A-F]+):", line)
        if cur is None or not m:
            continue
        goes = re.search(r"<(\S+?)(?:\+0x([0-9a-f]+))?>$", line)
        to = start[goes[1]] + int(goes[2] or "0", 16) if goes and m[1].startswith(("s_branch", "s_cbranch")) else None
        operands = [t.strip() for t in re.split(r",\s*(?![^\[]*\])", m[2].strip())] if m[2].strip() else []
        cur.append((int(m[3], 16), m[1], operands, to))
    return out


def first_touch(code, at, i):
    """(least number of slots, instruction) from matrix instruction i to what touches its result, over all paths; None: no such
    within MOST.  A matrix instruction that goes on from the result as its own addend waits by itself."""
    result = registers(code[i][2][0])
    best, todo, seen = None, [(i + 1, 0)], {}
    while todo:
        j, slots = todo.pop()
        while j < len(code) and slots < (best[0] if best else MOST) and seen.get(j, MOST) > slots:
            seen[j] = slots
            _, op, operands, to = code[j]
            if op in ("s_endpgm", "s_setpc_b64"):
                break
            if "mfma" in op:
                if (registers(operands[1]) | registers(operands[2])) & result:
                    best = (slots, " ".join([op] + operands))
                    break
                if registers(operands[0]) == result:
                    break  # its own result from here on
            elif not op.startswith("s_") and set().union(*map(registers, operands), set()) & result:
                best = (slots, " ".join([op] + operands))
                break
            slots += int(operands[0], 0) + 1 if op == "s_nop" else 1
            if to is not None:
                if op == "s_branch":
                    j = at[to]
                    continue
                todo.append((at[to], slots))
            j += 1
    return best


def waits(text):
    """opcode -> [(slots, function, what touches the result)]"""
    out = {}
    for name, code in functions(text).items():
        at = {c[0]: i for i, c in enumerate(code)}
        for i, c in enumerate(code):
            if "mfma" in c[1]:
                out.setdefault(c[1], [])
                hit = first_touch(code, at, i)
                if hit:
                    out[c[1]].append((hit[0], name, hit[1]))
    return out


@pytest.fixture(scope="module")
def disassemble(tmp_path_factory):
    if not (os.path.exists(OBJDUMP) and os.path.exists(HIPCC)):
        pytest.skip("no ROCm toolchain")

    def run(path):
        return subprocess.run([OBJDUMP, "-d", path], check=True, capture_output=True, text=True).stdout
    return run


@pytest.fixture(scope="module")
def needed(disassemble, tmp_path_factory):
    d = tmp_path_factory.mktemp("straight")
    (d / "s.hip").write_text(STRAIGHT)
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "--cuda-device-only", "--no-gpu-bundle-output", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-c", "-o", str(d / "s.o"), str(d / "s.hip")],
                   check=True, capture_output=True)
    text = disassemble(str(d / "s.o"))
    got = {op: min(hits)[0] for op, hits in waits(text).items()}
    assert len(got) == 4 and all(n >= 4 for n in got.values()), got
    for name, code in functions(text).items():  # (filled up to the slot: the number is the compiler's requirement and no accident)
        i = next(i for i, c in enumerate(code) if "mfma" in c[1])
        assert any(c[1] == "s_nop" for c in code[i + 1:i + 4]), name
    return got


def test_the_walk_sees_a_lost_wait():
    """(a listing made up for it: a read one slot behind a branch, beside a path that waits long enough)"""
    text = """
0000000000001000 <kernel>:
\tv_mfma_f32_16x16x32_bf16 v[4:7], v[8:11], v[12:15], v[4:7]// 000000001000: 0
\ts_cbranch_scc1 2                                           // 000000001008: 0 <kernel+0x14>
\ts_nop 7                                                    // 00000000100C: 0
\ts_nop 3                                                    // 000000001010: 0
\tv_add_f32_e32 v0, v1, v6                                   // 000000001014: 0
\ts_endpgm                                                   // 000000001018: 0
"""
    assert waits(text) == {"v_mfma_f32_16x16x32_bf16": [(1, "kernel", "v_add_f32_e32 v0 v1 v6")]}
    assert waits(text.replace("s_cbranch_scc1 2 ", "s_nop 2 ").replace(" <kernel+0x14>", ""))["v_mfma_f32_16x16x32_bf16"][0][0] == 3 + 8 + 4


def test_every_path_of_the_shipped_kernels_waits(disassemble, needed, tmp_path):
    if not os.path.exists(LIB):
        pytest.skip("the library is not built")
    shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    parts = sorted(p for p in os.listdir(tmp_path) if "amdgcn" in p)
    assert parts
    seen = 0
    for part in parts:
        for op, hits in waits(disassemble(str(tmp_path / part))).items():
            assert op in needed, f"{op}: add it to the straight lines"
            for slots, name, what in hits:
                assert slots >= needed[op], f"{name}: {what} stands {slots} slots behind a {op}, which takes {needed[op]}"
            seen += len(hits)
    assert seen > 100
