"""The many-row kernel issues v_mfma_f32_32x32x16_bf16 from inline asm, so the
compiler inserts no wait states around it. This compiles the kernels to
assembly and follows the registers along every path: two wait states between
a VALU write of an operand and the MFMA that reads it, and the pipe's 18
between an MFMA and a read or write of its result by anything but the next
MFMA on the same accumulators (11 for the 16x16x32 form). Scratch memory, which
cost 10 us a call where it was used, has to stay unused."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    if not Path(HIPCC).exists():
        pytest.skip("no hipcc")
    make = subprocess.run(["make", "-n", "-B", "_build/ops_k_attention_paged.o"],
                          cwd=ROOT / "cu-jev_amd", capture_output=True, text=True, check=True)
    line = next(x for x in make.stdout.splitlines() if "attention_paged.hip" in x)
    out = tmp_path_factory.mktemp("asm") / "attention_paged.s"
    args = re.sub(r"\s-c\s", " --cuda-device-only -S ", re.sub(r"-o \S+", f"-o {out}", line)).split()
    subprocess.run(args, cwd=ROOT / "cu-jev_amd", check=True, capture_output=True)
    return out.read_text()


def kernels(text):
    for m in re.finditer(r"^(_Z\S*kernel\S*):\s*;\s*@", text, re.M):
        yield m[1], text[m.end():text.index(".section", m.end())].splitlines()[1:]


def registers(operand):
    m = re.match(r"-?\|?([av])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.match(r"-?\|?([av])(\d+)\b", operand)
    return {(m[1], int(m[2]))} if m else set()


def instructions(lines):
    out = []
    for line in lines:
        line = line.split(";")[0].strip()
        if line.endswith(":"):
            out.append(("label", [line[:-1]]))
        elif line and not line.startswith("."):
            op, _, rest = line.partition(" ")
            out.append((op, [o.strip() for o in rest.split(",")] if rest else []))
    return out


def violations(code):
    """[(index, what)] where an operand or result comes too early on some path.
    State before an instruction: register -> wait states that are left, of VALU
    writes for MFMAs (0) and of MFMA results for the others (1)."""
    labels = {ops[0]: k for k, (op, ops) in enumerate(code) if op == "label"}
    before, work, bad = {0: ({}, {})}, [0], {}
    while work:
        k = work.pop()
        if k >= len(code):
            continue
        op, ops = code[k]
        valu, mfma = before[k]
        waits = 0 if op == "label" else int(ops[0], 0) + 1 if op == "s_nop" else 1
        is_mfma, is_valu = op.startswith("v_mfma"), op.startswith("v_")
        memory = op.startswith(("ds_", "buffer_", "global_", "scratch_"))
        if is_mfma:
            read = set().union(*map(registers, ops[1:4]))
            early = {r for r in read if r in valu}
            result = registers(ops[0])
            fresh = read if registers(ops[3]) != result else read - result
            early |= {r for r in fresh if r in mfma}
        else:
            early = {r for o in ops for r in registers(o) if r in mfma} \
                if is_valu or memory else set()
        if early:
            bad[k] = f"{op} {', '.join(ops)}: {sorted(early)[:4]}"
        valu = {r: v - waits for r, v in valu.items() if v > waits}
        # the next MFMA waits for the pipe, 8 passes of the one before
        step = 7 if is_mfma else waits
        mfma = {r: v - step for r, v in mfma.items() if v > step}
        if is_mfma:
            for r in result:
                mfma[r] = 19 if "32x32" in op else 11
                valu.pop(r, None)
        elif is_valu:
            for o in ops[:2 if "swap" in op else 1]:
                for r in registers(o):
                    valu[r] = 2
                    mfma.pop(r, None)
        elif op.startswith(("ds_read", "ds_bpermute", "buffer_load", "global_load")) and ops:
            for r in registers(ops[0]):
                valu.pop(r, None)
                mfma.pop(r, None)
        after = [] if op in ("s_endpgm", "s_setpc_b64") else \
            [labels[ops[0]]] if op == "s_branch" else \
            [k + 1, labels[ops[0]]] if op.startswith("s_cbranch") else [k + 1]
        for n in after:
            if n not in before:
                before[n] = (dict(valu), dict(mfma))
                work.append(n)
                continue
            grown = False
            for have, new in zip(before[n], (valu, mfma)):
                for r, v in new.items():
                    if have.get(r, 0) < v:
                        have[r], grown = v, True
            if grown:
                work.append(n)
    return sorted(bad.items())


def test_the_check_finds_what_it_is_for():
    def code(*lines):
        return instructions(list(lines) + ["s_endpgm"])

    mfma = "v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], a[0:3], v[0:15]"
    assert violations(code("v_mov_b32_e32 v20, v40", mfma))
    assert violations(code("v_mov_b32_e32 v20, v40", "s_nop 0", mfma))
    assert not violations(code("v_mov_b32_e32 v20, v40", "s_nop 1", mfma))
    assert not violations(code(mfma, mfma))
    assert violations(code(mfma, "s_nop 15", "v_add_f32_e32 v1, v1, v2"))
    assert not violations(code(mfma, "s_nop 15", "s_nop 7", "v_add_f32_e32 v1, v1, v2"))
    assert violations(code(mfma, "s_cbranch_scc1 .L", "s_nop 15", "s_nop 7", ".L:",
                           "v_add_f32_e32 v1, v1, v2"))


def test_mfmas_have_their_wait_states(assembly):
    seen = 0
    for name, lines in kernels(assembly):
        if "attention_many_kernel" not in name:
            continue
        code = instructions(lines)
        seen += sum("32x32x16" in op for op, _ in code)
        bad = violations(code)
        assert not bad, (name, bad[:4])
    assert seen >= 2 * 64


def test_no_scratch_memory(assembly):
    sizes = re.findall(r"ScratchSize: (\d+)", assembly)
    assert sizes and set(sizes) == {"0"}
