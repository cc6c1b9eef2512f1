"""No instruction of the kernels over heads reads a matrix product before it is
there (CPU only: the kernels are compiled to assembly, not run).

The hardware does not hold back a VALU or memory instruction that reads (or
overwrites) the result of a matrix instruction in flight; the compiler adds the
wait. Where a branch stood between the two it was found not to, and stale
accumulators were read. This follows every path from each v_mfma of the compiled
kernels, counting wait states (an instruction is one, s_nop n is n + 1), and asks
for the twelve that a 32x32x16 instruction takes (eight passes and four).
"""

from __future__ import annotations

import importlib.util
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "topk-tarmac_amd"
SOURCES = [f"mha_{way}_{dtype}" for way in ("fwd", "bwd") for dtype in ("f32", "bf16", "f16")]
WAIT_STATES = {"32x32x16": 12}


def _build():
    spec = importlib.util.spec_from_file_location("tarmac_build", PKG / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _registers(text: str) -> set[int]:
    regs = set()
    for lo, hi, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        regs |= {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return regs


def _functions(asm: str):
    """(name, instructions, label -> index) of each function."""
    name, code, labels = None, [], {}
    for line in asm.split("\n"):
        start = re.match(r"^(_Z\w+):", line)
        if start:
            name, code, labels = start.group(1), [], {}
        elif line.startswith(".Lfunc_end") and name:
            yield name, code, labels
            name = None
        elif name:
            label = re.match(r"^(\.LBB\w+):", line)
            text = line.split(";")[0].strip()
            if label:
                labels[label.group(1)] = len(code)
            elif text and not text.startswith("."):
                code.append(text)


def _next(code, labels, i):
    op, _, rest = code[i].partition(" ")
    if op == "s_endpgm":
        return []
    if op == "s_branch":
        return [labels[rest.strip()]]
    if op.startswith("s_cbranch"):
        return [i + 1, labels[rest.strip()]]
    return [i + 1]


def early_reads(asm: str):
    found, products = [], 0
    for name, code, labels in _functions(asm):
        for i, text in enumerate(code):
            if not text.startswith("v_mfma"):
                continue
            products += 1
            need = WAIT_STATES[re.search(r"_(\d+x\d+x\d+)_", text).group(1)]
            result = _registers(text.split(None, 1)[1].split(",")[0])
            best, todo = {}, [(j, 0) for j in _next(code, labels, i)]
            while todo:
                j, waited = todo.pop()
                if waited >= need or best.get(j, need) <= waited:
                    continue
                best[j] = waited
                op, _, rest = code[j].partition(" ")
                if op.startswith("v_mfma"):
                    operands = [x.strip() for x in re.split(r",(?![^\[]*\])", rest)]
                    if (_registers(operands[1]) | _registers(operands[2])) & result:
                        found.append((name, text, code[j], waited))
                    if _registers(operands[0]) & result:
                        continue  # accumulates on: its own result is followed from there
                elif not op.startswith("s_") and _registers(rest) & result:
                    found.append((name, text, code[j], waited))
                    continue
                waited += int(rest.strip(), 0) + 1 if op == "s_nop" else 1
                todo += [(k, waited) for k in _next(code, labels, j)]
    return found, products


def test_the_scan_finds_an_early_read():
    asm = "\n".join(["_Zk:", "\tv_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], 0", "\ts_cbranch_scc1 .LBB0_2",
                     "\ts_nop 11", ".LBB0_2:", "\tv_add_f32_e32 v30, v31, v15", "\ts_endpgm", ".Lfunc_end0:"])
    found, products = early_reads(asm)
    assert products == 1 and [f[3] for f in found] == [1]
    found, _ = early_reads(asm.replace("\ts_cbranch_scc1 .LBB0_2\n", ""))
    assert not found


def _assembly(source: str, out: Path) -> str:
    b = _build()
    run = subprocess.run([b.hipcc(), *b.HIPCC_FLAGS, "--cuda-device-only", "-S", str(b.CSRC / f"{source}.hip"), "-o",
                          str(out / f"{source}.s")], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    return (out / f"{source}.s").read_text()


@pytest.mark.timeout(600)
def test_no_product_is_read_early(tmp_path):
    with ThreadPoolExecutor(max_workers=6) as pool:
        for source, asm in zip(SOURCES, pool.map(lambda s: _assembly(s, tmp_path), SOURCES)):
            found, products = early_reads(asm)
            assert products > 100, source
            assert not found, (source, len(found), found[:3])
            # nor does a kernel keep registers in memory
            for name, size in re.findall(r"\.name:\s+(\S+)\n(?:.*\n)*?\s+\.private_segment_fixed_size:\s+(\d+)", asm):
                assert size == "0", (source, name, size)
