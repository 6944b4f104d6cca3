"""No instruction of the built kernels touches a matrix result before its wait states have passed.

A matrix instruction's result may be read or overwritten by another unit some wait states after
it at the earliest (every instruction is one, ``s_nop n`` is n + 1).  The compiler inserts them, but
where a branch skips a block of products it counts along the way through that block only, so the
kernels wait on the way around by themselves.  Counted here on the machine code of this
repository's own kernels, over every path.
"""

from __future__ import annotations

import re
import subprocess
from collections import defaultdict
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "hexo-shrimp-bot_amd"
ROCM = Path("/opt/rocm")
OBJDUMP = ROCM / "llvm" / "bin" / "llvm-objdump"
LINE = re.compile(r"^\s+([a-z]\S*)\s*(.*?)\s*// ([0-9A-F]+): (.*)$")
REGS = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")
# gfx950, as the compiler itself keeps them in straight-line code
STATES = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x4_f32": 10,
          "v_mfma_f32_4x4x1_16b_f32": 4}

pytestmark = pytest.mark.skipif(not OBJDUMP.exists(), reason="no disassembler")


def _regs(text):
    out = set()
    for kind, lo, hi, one in REGS.findall(text):
        out.update((kind, i) for i in range(int(lo or one), int(hi or one) + 1))
    return out


def _kernels(text):
    """(name, instructions) of every kernel that multiplies matrices: (address, words, mnemonic, operands)."""
    for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
        if "v_mfma" not in part:
            continue
        name = part[part.index("<") + 1:part.index(">:")]
        code = []
        for line in part.splitlines()[1:]:
            m = LINE.match(line)
            if m:
                code.append((int(m[3], 16), len(m[4].split("<")[0].split()), m[1], m[2]))
        yield name, code


def _least_states(code):
    """{matrix instruction: (fewest wait states before its result is touched, where)} over every path."""
    at = {addr: i for i, (addr, *_rest) in enumerate(code)}

    def after(i):
        addr, words, op, args = code[i]
        if op == "s_endpgm":
            return []
        if op.startswith(("s_cbranch", "s_branch")):
            to = at[addr + 4 + 4 * ((int(args.split()[0]) + 0x8000) % 0x10000 - 0x8000)]
            if op == "s_cbranch_execz" and not idle[i]:
                return [i + 1]  # (the compiler's form of a branch that is never taken)
            return [to] if op == "s_branch" else [to, i + 1]
        return [i + 1]

    # where the wavefront may have no lane: from a narrowed mask on, until it is tested or widened again
    idle, todo = [False] * len(code), [(0, False)]
    reached = [False] * len(code)
    while todo:
        i, none = todo.pop()
        while not (reached[i] and (idle[i] or not none)):
            reached[i], idle[i] = True, idle[i] or none
            _, _, op, args = code[i]
            if "saveexec" in op or re.match(r"s_(and|andn2|xor)\w* exec,", f"{op} {args}"):
                none = True
            elif re.match(r"s_(or|mov)\w* exec,", f"{op} {args}"):
                none = False
            ways = after(i)
            if not ways:
                break
            if op == "s_cbranch_execz" and len(ways) == 2:
                todo.append((ways[0], True))
                i, none = ways[1], False
            else:
                todo.extend((w, none) for w in ways[1:])
                i = ways[0]

    least = {}
    for i, (_addr, _words, op, args) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        result = _regs(args.split(", ")[0])
        need = STATES[op]
        todo, seen = [(j, 0) for j in after(i)], {}
        while todo:
            j, states = todo.pop()
            if states >= need or seen.get(j, need) <= states or j >= len(code):
                continue
            seen[j] = states
            _, _, other, operands = code[j]
            if other.startswith("v_mfma"):
                d, a, b, c = (_regs(x) for x in operands.split(", ")[:4])
                if (a | b) & result:
                    least[op] = min(least.get(op, (need, "")), (states, f"{code[i]} -> {code[j]}"))
                if (d | c) & result:  # summed on, or written anew: that one's result from there
                    continue
            elif not other.startswith("s_") and _regs(operands) & result:
                least[op] = min(least.get(op, (need, "")), (states, f"{code[i]} -> {code[j]}"))
                continue
            states += int(operands, 0) + 1 if other == "s_nop" else 1
            todo.extend((k, states) for k in after(j))
    return least


def _check(objects):
    kernels, bad = 0, defaultdict(list)
    for text in objects:
        for name, code in _kernels(text):
            kernels += 1
            for op, found in _least_states(code).items():
                bad[name].append((op, *found))
    assert not bad, dict(bad)
    return kernels


def _disassembled(obj):
    return subprocess.run([str(OBJDUMP), "-d", str(obj)], capture_output=True, text=True, check=True).stdout


def test_the_count_sees_an_early_reader():
    line = "\t{} // {:012X}: 00000000 00000000\n"

    def code(gap):
        ops = ["v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]", "s_cbranch_scc1 3", "s_nop 7", f"s_nop {gap}",
               "v_add_f32_e32 v9, v2, v9", "s_endpgm"]
        return next(_kernels("0000000000000000 <k>:\n" + "".join(line.format(op, 8 * i) for i, op in enumerate(ops))))[1]

    # (s_cbranch at 8 jumps to 12 + 4 * 3 = 24, past the first s_nop)
    assert _least_states(code(5))["v_mfma_f32_16x16x32_bf16"][0] == 7
    assert not _least_states(code(6))


def test_built_kernels(tmp_path):
    lib = tmp_path / "libmantis_hip.so"
    lib.symlink_to(PKG / "libmantis_hip.so")
    subprocess.run([str(OBJDUMP), "--offloading", lib.name], cwd=tmp_path, check=True, capture_output=True)
    kernels = _check(_disassembled(x) for x in sorted(tmp_path.glob("*gfx950*")))
    assert kernels > 100, kernels


def test_relative_attention_with_results_in_accumulators(tmp_path):
    """The waits belong to the source, not to where the build's flags keep the results."""
    obj = tmp_path / "relative_attention.o"
    subprocess.run([str(ROCM / "bin" / "hipcc"), "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature",
                    "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "--no-gpu-bundle-output", "-c",
                    str(PKG / "csrc" / "kernels" / "relative_attention.hip"), "-o", str(obj)], check=True,
                   capture_output=True)
    assert _check([_disassembled(obj)])
