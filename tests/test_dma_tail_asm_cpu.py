"""The direct-to-LDS GEMM kernels (gemm_dma.h) read LDS fragments by inline asm and wait for them themselves.  The
last reads of the main loop land in registers nobody uses.  Until they are waited for, nothing else may be written
to those registers: a read that lands late would overwrite it (address arithmetic of the epilogue: a wild store).
The gfx950 code objects of the built library are disassembled; no GPU is needed."""
from __future__ import annotations

import re
import subprocess
import tempfile

import pytest

from tests.test_agpr_asm_cpu import _code_objects, _tool

KERNEL = re.compile(r"_ZN3skl15gemm_dma_kernel\S*")


def _kernels():
    objdump = _tool("llvm-objdump")
    if not objdump:
        pytest.skip("llvm-objdump is not available")
    kernels = {}
    with tempfile.TemporaryDirectory() as d:
        for co in _code_objects(d):
            table = subprocess.run([objdump, "-t", co], check=True, capture_output=True, text=True).stdout
            syms = sorted({m.group(0) for m in KERNEL.finditer(table) if not m.group(0).endswith(".kd")})
            if not syms:
                continue
            out = subprocess.run([objdump, "-d", "--mcpu=gfx950", "--disassemble-symbols=" + ",".join(syms), co],
                                 check=True, capture_output=True, text=True).stdout
            cur = None
            for line in out.splitlines():
                m = re.match(r"^[0-9a-f]+ <(\S+)>:", line)
                if m:
                    cur = kernels.setdefault(m.group(1), [])
                elif cur is not None and line.startswith("\t"):
                    cur.append(line.strip().split("//")[0].strip())
    return kernels


def _vgprs(operand):
    m = re.match(r"v\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.match(r"v(\d+)\b", operand)
    return {int(m.group(1))} if m else set()


def _first_operand(ins):
    parts = ins.split(None, 1)
    return parts[1].split(",")[0].strip() if len(parts) == 2 else ""


def test_nothing_is_written_to_registers_of_reads_in_flight():
    kernels = _kernels()
    assert len(kernels) >= 20
    seen = 0
    for name, ins in kernels.items():
        last = max(i for i, s in enumerate(ins) if s.startswith("v_mfma"))
        full = [i for i, s in enumerate(ins[:last]) if "lgkmcnt(0)" in s]
        flying = {}
        for s in ins[full[-1] + 1:last + 1]:
            if s.startswith("ds_read"):
                flying |= {r: s for r in _vgprs(_first_operand(s))}
        for s in ins[last + 1:]:
            if "lgkmcnt(0)" in s:
                break
            if s.startswith("ds_read"):
                flying |= {r: s for r in _vgprs(_first_operand(s))}
            elif not s.startswith(("ds_write", "global_store", "buffer_store", "s_")):
                hit = _vgprs(_first_operand(s)) & set(flying)
                assert not hit, f"{name}: '{s}' writes registers of '{flying[min(hit)]}' in flight"
        seen += bool(flying)
    assert seen >= 20, "no reads in flight found: the kernels' last reads look otherwise now"
