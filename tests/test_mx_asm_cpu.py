"""The tiled 4-bit product issues its MFMAs from inline asm, where the compiler's hazard checks do not
look.  On the code of the built library (no GPU needed), for every such kernel:

  * between the first and the last MFMA nothing else writes an AGPR, and the zeroing before the first
    is 2 wait states away from it;
  * what first touches an AGPR behind the last MFMA is 19 wait states away;
  * no VALU instruction writes a fragment or scale register less than 2 wait states before the MFMA
    that reads it.
"""
from __future__ import annotations

import re

from tests import test_agpr_asm_cpu as asm

KERNEL = re.compile(r"_ZN3skl14mx_gemm_kernel\S*")


def registers(operand):
    m = re.fullmatch(r"v(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    return {int(m.group(1))} if m.group(1) else set(range(int(m.group(2)), int(m.group(3)) + 1))


def operands(ins):
    parts = ins.split(None, 1)
    return [p.split()[0] for p in parts[1].split(",") if p.strip()] if len(parts) == 2 else []


def test_the_asm_products_wait_states(monkeypatch):
    monkeypatch.setattr(asm, "ONE_WAVE", KERNEL)
    kernels = asm._disassembly()
    assert len(kernels) == 4, sorted(kernels)   # two types, two tiles
    for name, ins in kernels.items():
        mfma = [i for i, s in enumerate(ins) if s.startswith("v_mfma")]
        tiles = 32 if "Li256E" in name else 16
        assert len(mfma) >= 2 * tiles and all("v_mfma_scale_f32_16x16x128" in ins[i] for i in mfma), name
        first, last = mfma[0], mfma[-1]
        bad = [s for s in ins[first:last + 1] if asm._writes_agpr(s) and not s.startswith("v_mfma")]
        assert not bad, f"{name}: AGPR written between MFMAs by {bad[:3]}"
        zero = [i for i, s in enumerate(ins[:first]) if s.startswith("v_accvgpr_write")]
        assert zero and asm._wait_states(ins[zero[-1] + 1:first]) >= 2, f"{name}: zeroing too close to the first MFMA"
        reads = [i for i, s in enumerate(ins) if i > last and re.search(r"\ba(\d+|\[\d+:\d+\])", s)]
        assert reads and asm._wait_states(ins[last + 1:reads[0]]) >= 19, f"{name}: sums read too soon"
        for i in mfma:
            ops = operands(ins[i])
            sources = set().union(*(registers(o) for o in ops[1:]))
            assert len(sources) == 10, ins[i]   # two fragments of 4 and two scales
            j, waited = i - 1, 0
            while j >= 0 and waited < 2:
                s = ins[j]
                if s.startswith("v_") and not s.startswith(("v_mfma", "v_nop")):
                    assert not (registers(operands(s)[0]) & sources), f"{name}: {s} before {ins[i]}"
                waited += asm._wait_states([s])
                j -= 1
