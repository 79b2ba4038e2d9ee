"""The built kernels wait for their matrix instructions.

A matrix instruction writes its result some cycles after it issues, and nothing but instructions in between (or s_nop)
keeps a later one from reading the registers before: 8 of them behind a 16-bit product of 16 x 16 x 32, 10 behind a float
one of 16 x 16 x 4, which is what the compiler puts there in straight code.  Behind a branch that is taken it has been
seen to put none (a uniform branch between a product and the first use of its result); sources keep branches
away from there, and this test looks through the disassembly of the built library along every path."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

LIBRARY = Path(__file__).resolve().parent.parent / "relmo_amd" / "librelm_mp_hip.so"
OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
WAITS = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x4_f32": 10}
OPERAND = re.compile(r"^[-|]*([va])(?:(\d+)|\[(\d+):(\d+)\])")


def _registers(operands) -> set:
    found = set()
    for text in operands:
        m = OPERAND.match(text)
        if m:
            first, last = (m[2], m[2]) if m[2] else (m[3], m[4])
            found.update((m[1], n) for n in range(int(first), int(last) + 1))
    return found


def _instructions(listing: str):
    code, labels, name = [], {}, ""
    for line in listing.splitlines():
        if line.startswith("<"):
            label = line[1:line.rindex(">")]
            name = name if re.fullmatch(r"L\d+", label) else label
            labels[label] = len(code)
        elif line.startswith("\t"):
            op, _, rest = line.split("//")[0].strip().partition(" ")
            code.append((op, [o.strip() for o in re.split(r",\s*(?![^\[]*\])", rest)] if rest.strip() else [], name))
    return code, labels


def early_reads(listing: str) -> list:
    code, labels = _instructions(listing)
    found, unknown = [], set()
    for at, (op, operands, name) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        if op not in WAITS:
            unknown.add(op)
            continue
        result, need, paths, seen = _registers(operands[:1]), WAITS[op], [(at + 1, 0)], {}
        while paths:
            i, waited = paths.pop()
            while i < len(code) and waited < need and seen.get(i, need) > waited:
                seen[i] = waited
                o, args, _ = code[i]
                if o == "s_endpgm":
                    break
                if o == "s_nop":
                    waited += int(args[0], 0)
                elif o == "s_branch":
                    i = labels[args[0]] - 1
                elif o.startswith("s_cbranch"):
                    paths.append((labels[args[0]], waited + 1))
                elif o.startswith("v_mfma"):
                    if _registers(args[1:3]) & result:  # as a factor; added to, it is forwarded
                        found.append((name, op, o, args, waited))
                        break
                    if _registers(args[:1]) >= result:
                        break
                elif _registers(args) & result:
                    found.append((name, op, o, args, waited))
                    break
                waited += 1
                i += 1
    assert not unknown, unknown
    return found


def _listings(library: Path, folder: Path):
    shutil.copy(library, folder / "library.so")
    subprocess.run([OBJDUMP, "--offloading", "library.so"], cwd=folder, check=True, capture_output=True)
    for part in sorted(folder.glob("library.so.*gfx950*")):
        yield subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", "--symbolize-operands", part], check=True,
                             capture_output=True, text=True).stdout


def test_results_of_matrix_instructions_are_waited_for(tmp_path) -> None:
    if not LIBRARY.exists() or not OBJDUMP.exists():
        pytest.skip("needs the built library and llvm-objdump")
    products = 0
    for listing in _listings(LIBRARY, tmp_path):
        products += listing.count("v_mfma")
        found = early_reads(listing)
        assert not found, (len(found), found[:5])
    assert products > 10_000


def test_the_scan_sees_a_read_behind_a_taken_branch() -> None:
    def listing(nops: int) -> str:
        return ("<kernel>:\n\tv_mfma_f32_16x16x32_f16 v[2:5], v[6:9], v[10:13], 0 // 0\n\ts_cbranch_vccz L1 // 8\n"
                f"\ts_nop 7 // c\n<L1>:\n\ts_nop {nops} // 10\n\tv_fma_f32 v1, v4, v20, -v21 // 14\n\ts_endpgm // 1c\n")

    assert len(early_reads(listing(5))) == 1 and not early_reads(listing(6))
