"""CPU test of csrc/fq_dma.h's copies, on the assembly that the compiler makes of them.

A vector-memory instruction must not read a scalar register within five states of the vector
instruction that wrote it.  The compiler sees to that for its own instructions, not
for those in inline assembly, so the copies have to wait by themselves."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from forge_amd import build

SOURCE = """
#include "fq_dma.h"
// the base, and then the place in LDS, are made uniform right before the copy
extern "C" __global__ void base_from_a_lane(const uint8_t* const* p, float* out) {
    extern __shared__ uint8_t lds[];
    const uint64_t at = (uint64_t)p[threadIdx.x];
    const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
    fq::dma16s(16 * threadIdx.x, (const uint8_t*)base, fq::lds_addr(lds));
    fq::wait_vm<0>();
    out[threadIdx.x] = *(float*)(lds + 16 * threadIdx.x);
}
extern "C" __global__ void place_from_a_lane(const uint8_t* p, const int* at, float* out) {
    extern __shared__ uint8_t lds[];
    fq::dma16s(16 * threadIdx.x, p, (uint32_t)__builtin_amdgcn_readfirstlane(at[threadIdx.x]));
    fq::wait_vm<0>();
    out[threadIdx.x] = *(float*)(lds + 16 * threadIdx.x);
}
"""


def registers(text):
    """The scalar registers that an operand list names."""
    regs = {"m0"} if re.search(r"\bm0\b", text) else set()
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        regs |= set(range(int(a), int(b) + 1))
    return regs | {int(a) for a in re.findall(r"\bs(\d+)\b", text)}


def too_early(asm):
    """The copies that read a register a vector instruction wrote less than five states before."""
    found, copies, past = [], 0, []
    for line in asm.splitlines():
        line = line.split(";")[0].strip()
        if re.match(r"^\w+:$", line):
            past = []
        if not line or line.startswith((".", "#")) or line.endswith(":"):
            continue
        op, _, args = line.partition(" ")
        if op.startswith("global_load_lds"):
            copies += 1
            reads, states = registers(args) | {"m0"}, 0
            for before, its in reversed(past):
                if states >= 5:
                    break
                wrote = registers(its.split(",")[0])
                if before.startswith("v_") and wrote & reads:
                    found.append((before, its, line, states))
                if before.startswith("s_"):  # (which waits for what vector instructions wrote)
                    reads -= wrote
                states += int(its, 0) + 1 if before == "s_nop" else 1
        past.append((op, args.strip()))
    return copies, found


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="needs hipcc")
def test_copies_wait_for_registers_that_vector_instructions_wrote(tmp_path):
    src, out = tmp_path / "dma.hip", tmp_path / "dma.s"
    src.write_text(SOURCE)
    subprocess.run([build.HIPCC, *build.COMMON, "-I", build.CSRC, "--offload-device-only", "-S", str(src),
                    "-o", str(out)], check=True, capture_output=True)
    copies, found = too_early(out.read_text())
    assert copies == 2
    assert not found, found
