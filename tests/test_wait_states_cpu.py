"""Wait states between a matrix instruction and the first instruction that touches its result, on EVERY path of the built code.

The hardware does not interlock these: the compiler inserts ``s_nop``.  hipcc (ROCm 7.2) leaves them out now and then where a branch
stands between the two -- it counts one path and the other is shorter -- and the first read behind the branch then sees the last row
of the 32 x 32 tile before it was written.  No parity test shows it reliably (whether another wave's instructions happen to fill the
gap depends on the launch), so this one walks the control-flow graph of the disassembled object that ``__graft_entry__.build()`` left
in ``csrc/obj``.  Distances are those hipcc uses where no branch intervenes: 12 for v_mfma_f32_32x32x16_bf16, 18 for
v_mfma_f32_32x32x2_f32."""

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LLVM = "/opt/rocm/lib/llvm/bin"
NEEDED = {"v_mfma_f32_32x32x16_bf16": 12, "v_mfma_f32_32x32x2_f32": 18}
LOADS = ("ds_read", "global_load", "buffer_load", "scratch_load")


def disassemble(unit, work):
    tools = [os.path.join(LLVM, t) for t in ("llvm-objcopy", "clang-offload-bundler", "llvm-objdump")]
    built = os.path.join(ROOT, "kronfluence_amd", "csrc", "obj", unit + ".o")
    if not os.path.exists(built) or not all(os.path.exists(t) for t in tools):
        pytest.skip("needs the object files of __graft_entry__.build() and the ROCm LLVM tools")
    fat, code, local = (str(work / n) for n in ("fat.bin", "device.co", unit + ".o"))
    shutil.copy(built, local)   # llvm-objcopy rewrites its input when asked to dump a section
    subprocess.run([tools[0], "--dump-section", f".hip_fatbin={fat}", local], check=True)
    subprocess.run([tools[1], "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={fat}", f"--output={code}"],
                   check=True)
    text = subprocess.run([tools[2], "-d", "--no-show-raw-insn", code], check=True, capture_output=True, text=True).stdout.splitlines()
    heads = [i for i, line in enumerate(text) if re.match(r"^[0-9a-f]+ <", line)] + [len(text)]
    for begin, end in zip(heads, heads[1:]):
        body = []
        for line in text[begin + 1:end]:
            m = re.match(r"^\s+(\S+)\s*(.*?)\s*//\s*([0-9A-F]+):", line)
            if m:
                target = re.search(r"\+0x([0-9a-f]+)>", line)
                body.append((int(m.group(3), 16), m.group(1), m.group(2), int(target.group(1), 16) if target else None))
        if body:
            yield re.search(r"<(.*)>:", text[begin]).group(1), body


def registers(operands):
    found = set()
    for kind, first, last, one in re.findall(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+))", operands):
        found.update((kind, i) for i in (range(int(first), int(last) + 1) if not one else [int(one)]))
    return found


def violations(body):
    """(matrix instruction, the instruction that touches its result too early, wait states between them)"""
    base, index = body[0][0], {entry[0]: i for i, entry in enumerate(body)}
    for i, (_, op, operands, _) in enumerate(body):
        if op not in NEEDED:
            continue
        result = registers(operands.split(",")[0])
        paths, best = [(i + 1, 0)], {}
        while paths:
            at, waited = paths.pop()
            if at >= len(body) or waited >= NEEDED[op] or best.get(at, NEEDED[op]) <= waited:
                continue
            best[at] = waited
            _, other, args, target = body[at]
            if other == "s_endpgm":
                continue
            fields = args.split(",")
            if other.startswith("v_mfma"):      # (its accumulator operand is forwarded)
                touched = registers(",".join(fields[1:3]))
            elif other.startswith(LOADS):
                touched = registers(",".join(fields[1:]))
            else:
                touched = set() if other.startswith("s_") else registers(args)
            if touched & result:
                yield f"{op} {operands}", f"{other} {args}", waited
                continue
            if other.startswith("v_mfma") and registers(fields[0]) >= result:
                continue
            if "branch" in other and target is not None and base + target in index:
                paths.append((index[base + target], waited + 1))
            if other != "s_branch":
                paths.append((at + 1, waited + 1 + (int(args) if other == "s_nop" else 0)))


@pytest.mark.parametrize("unit", ["kf_attention", "kf_kernels", "kf_score_v2"])
def test_results_of_matrix_instructions_are_not_touched_too_early(unit, tmp_path):
    kernels = 0
    for name, body in disassemble(unit, tmp_path):
        kernels += any(op in NEEDED for _, op, _, _ in body)
        assert not list(violations(body)), name
    assert kernels > 0


def test_the_walk_finds_the_shorter_path():
    """The pattern that was miscompiled: long enough in a straight line, too short where the branch is taken."""
    body = [(0, "v_mfma_f32_32x32x2_f32", "a[0:15], v0, v1, a[0:15]", None), (8, "s_cbranch_vccnz", "2", 16), (12, "s_nop", "12", None),
            (16, "s_nop", "3", None), (20, "v_accvgpr_read_b32", "v2, a15", None), (28, "s_endpgm", "", None)]
    assert [w for _, _, w in violations(body)] == [5]
    body[3] = (16, "s_nop", "15", None)
    body.insert(4, (18, "s_nop", "0", None))
    assert not list(violations(body))
