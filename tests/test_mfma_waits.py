"""A matrix instruction's result may be read, or its registers written, only some issue slots after it: the hardware does
not wait by itself, the compiler counts the instructions between. It has miscounted where a branch follows the last product
(the result was then read a few slots after it on the path that takes the branch, and the tokens of the last registers had
wrong scores), so the listing is counted here again, along every path.

The same listing is checked for scratch memory: no attention kernel spills registers."""

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "haskell-infer-demo_amd")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def registers(operand):
    m = re.match(r"-?\|?([va])\[(\d+):(\d+)\]", operand)
    if m:
        return {m.group(1) + str(i) for i in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.match(r"-?\|?([va])(\d+)\|?$", operand)
    return {m.group(1) + m.group(2)} if m else set()


def slots_needed(op):
    """Passes of the instruction (8, 4, 16) and four more, before another kind of instruction may touch its result."""
    return 12 if "32x32x16" in op else 8 if "16x16x32" in op else 20


def early_uses(asm):
    bad = []
    for m in re.finditer(r"^(_Z\w+):", asm, re.M):
        code, labels = [], {}
        for line in asm[m.end():asm.find(".Lfunc_end", m.end())].split("\n"):
            line = line.strip()
            label = re.match(r"(\.LBB\w+):", line)
            if label:
                labels[label.group(1)] = len(code)
            elif line and line[0] not in ";.":
                code.append(re.split(r"[ ,]+", line.split(";")[0].strip()))
        for i, t in enumerate(code):
            if not t[0].startswith("v_mfma"):
                continue
            result, paths, seen = registers(t[1]), [(i + 1, 0)], {}
            while paths:
                j, slots = paths.pop()
                if j >= len(code) or slots >= slots_needed(t[0]) or seen.get(j, 99) <= slots:
                    continue
                seen[j] = slots
                x = code[j]
                if x[0] == "s_nop":
                    paths.append((j + 1, slots + int(x[1]) + 1))
                    continue
                if x[0].startswith("v_mfma"):
                    # the same accumulator again is forwarded; as a factor it is not
                    if (registers(x[2]) | registers(x[3])) & result:
                        bad.append((m.group(1), " ".join(t), slots, " ".join(x)))
                        continue
                elif not x[0].startswith("s_") and any(registers(o) & result for o in x[1:]):
                    bad.append((m.group(1), " ".join(t), slots, " ".join(x)))
                    continue
                if x[0] == "s_endpgm":
                    continue
                if x[0].startswith(("s_branch", "s_cbranch")):
                    paths.append((labels[x[1]], slots + 1))
                if x[0] != "s_branch":
                    paths.append((j + 1, slots + 1))
    return bad


@pytest.fixture(scope="module")
def attention_asm(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc is not available")
    lines = subprocess.run(["make", "-n", "-B", "-C", PKG, "_build/attention.o"], check=True, capture_output=True, text=True).stdout
    command = next(line for line in lines.splitlines() if "attention.hip" in line).split()
    out = tmp_path_factory.mktemp("asm") / "attention.s"
    command = [HIPCC if c.endswith("hipcc") else c for c in command[:command.index("-c")]]
    subprocess.run(command + ["-S", "--cuda-device-only", "csrc/attention.hip", "-o", str(out)], check=True, capture_output=True, cwd=PKG)
    return out.read_text()


def test_results_are_waited_for(attention_asm):
    assert attention_asm.count("v_mfma") > 400
    assert early_uses(attention_asm) == []


def test_no_kernel_spills(attention_asm):
    sizes = re.findall(r"\.amdhsa_private_segment_fixed_size (\d+)", attention_asm)
    assert len(sizes) >= 18 and set(sizes) == {"0"}


def test_the_check_follows_branches():
    listing = """_Zk:
    v_mfma_f32_32x32x16_bf16 a[0:15], v[0:3], v[4:7], a[0:15]
    s_cbranch_vccnz .LBB0_2
    s_nop 15
.LBB0_2:
    s_nop 1
    v_accvgpr_read_b32 v9, a15
    s_endpgm
.Lfunc_end0:
_Zok:
    v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[4:7], v[0:3]
    v_mfma_f32_16x16x32_bf16 v[0:3], v[12:15], v[4:7], v[0:3]
    s_nop 7
    v_mul_f32_e32 v0, v1, v2
    s_endpgm
.Lfunc_end1:
"""
    assert [(name, slots) for name, _, slots, _ in early_uses(listing)] == [("_Zk", 3)]
