"""The DMAs to LDS of the 8-bit products are inline assembly, for which the
compiler does not keep the wait states that the hardware leaves to software:
five between a vector instruction that writes a scalar register and a vector
memory instruction that reads it, one between a write of m0 and a load to LDS.
These tests look for both in the assembly of the library as it was built."""
import os
import re
import shutil
import subprocess

import pytest

from shady_thinker_amd import build as hip_build

OBJDUMP = os.path.join(os.path.dirname(os.path.realpath(hip_build.HIPCC)), "..", "llvm", "bin", "llvm-objdump")
VCC = {"vcc": (106, 107), "vcc_lo": (106,), "vcc_hi": (107,)}
M0 = "m0"


def scalars(operand):
    """The scalar registers that an operand names."""
    operand = operand.strip()
    if operand in VCC:
        return set(VCC[operand])
    if operand == "m0":
        return {M0}
    m = re.fullmatch(r"s(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    return {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))


class Instruction:
    def __init__(self, text, target=None):
        self.name, _, rest = text.strip().partition(" ")
        ops = [o for o in re.split(r",\s*", rest.strip()) if o]
        self.text, self.target = text.strip(), target
        # (the last operand is followed by modifiers)
        ops = ops[:-1] + ops[-1].split()[:1] if ops else ops
        regs = [scalars(o) for o in ops]
        valu = self.name.startswith("v_")
        carry = valu and re.search(r"_co_|mad_[ui]64|div_scale", self.name)
        self.vector_writes = (regs[0] if valu and regs else set()) | (regs[1] if carry and len(regs) > 1 else set())
        if self.name.startswith("v_cmp") and not self.name.startswith("v_cmpx") and not self.vector_writes:
            self.vector_writes = {106, 107}  # (vcc, unnamed)
        scalar = self.name.startswith("s_") and not re.match(r"s_(cmp|bitcmp|cbranch|branch|waitcnt|nop|barrier|endpgm|setprio|sleep)", self.name)
        self.scalar_writes = regs[0] if scalar and regs else set()
        self.memory = self.name.startswith(("buffer_", "global_", "flat_", "scratch_"))
        self.to_lds = self.memory and (" lds" in self.text or "_lds_" in self.name)
        self.reads = set().union(*regs) if self.memory and regs else set()
        self.states = int(ops[0], 0) + 1 if self.name == "s_nop" else 1
        self.ends = self.name in ("s_branch", "s_endpgm", "s_setpc_b64")


def hazards(code):
    """{(instruction, the one it comes too soon after)} of a function."""
    before = [[i - 1] if i and not code[i - 1].ends else [] for i in range(len(code))]
    for i, c in enumerate(code):
        if c.target is not None:
            before[c.target].append(i)
    found = set()

    def back(i, reg, need, states, at):
        for j in before[i]:
            c = code[j]
            if reg in (c.scalar_writes if reg == M0 else c.vector_writes):
                found.add((at.text, c.text))
            elif reg not in c.scalar_writes and states + c.states < need:
                back(j, reg, need, states + c.states, at)

    for i, c in enumerate(code):
        for reg in c.reads:
            back(i, reg, 5, 0, c)
        if c.to_lds:
            back(i, M0, 1, 0, c)
    return found


def functions(listing):
    """{name: [Instruction]} of llvm-objdump's listing."""
    out = {}
    for part in re.split(r"^(?=[0-9a-f]{16} <)", listing, flags=re.M)[1:]:
        head, _, body = part.partition("\n")
        start, name = int(head[:16], 16), re.search(r"<(.*)>", head)[1]
        lines, at = [], {}
        for line in body.split("\n"):
            m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):", line)
            if m:
                at[int(m[2], 16)] = len(lines)
                to = re.search(r"<.*?\+0x([0-9a-f]+)>\s*$", line) if m[1].startswith(("s_cbranch", "s_branch")) else None
                lines.append((m[1], start + int(to[1], 16) if to else None))
        out[name] = [Instruction(text, at[to] if to is not None else None) for text, to in lines]
    return out


def listing_of(lines):
    """llvm-objdump's listing of a function of 4-byte instructions; (text, index
    it branches to)."""
    rows = []
    for i, line in enumerate(lines):
        text, to = line if isinstance(line, tuple) else (line, None)
        rows.append(f"\t{text}   // {4 * i:012X}: 00000000" + (f" <f+0x{4 * to:x}>" if to is not None else ""))
    return "0000000000000000 <f>:\n" + "\n".join(rows) + "\n"


LOAD = "buffer_load_dwordx4 v3, s[8:11], s5 offen lds"


@pytest.mark.parametrize("lines,bad", [
    (["v_readfirstlane_b32 s5, v0", "s_mov_b32 m0, s2", "s_nop 0", LOAD], 1),
    (["v_readfirstlane_b32 s5, v0", "s_mov_b32 m0, s2", "s_nop 3", LOAD], 0),
    (["v_readfirstlane_b32 s9, v0", "s_mov_b32 m0, s2", "s_nop 2", LOAD], 1),
    (["v_readlane_b32 s10, v0, 3", "s_mov_b32 m0, s2", "s_nop 0", LOAD], 1),
    (["v_readfirstlane_b32 s5, v0", "s_mov_b32 s5, s6", "s_mov_b32 m0, s2", "s_nop 0", LOAD], 0),
    (["v_add_co_u32_e64 v1, s[8:9], v1, v2", "s_mov_b32 m0, s2", "s_nop 0", LOAD], 1),
    (["v_cmp_eq_u32_e32 vcc, v1, v2", "s_mov_b32 m0, s2", "s_nop 0", LOAD.replace("s5", "vcc_lo")], 1),
    (["v_add_f32_e32 v5, s5, v1", "s_mov_b32 m0, s2", "s_nop 0", LOAD], 0),
    (["s_nop 7", "s_mov_b32 m0, s2", LOAD], 1),
    # at a loop's head, the write at its end
    (["s_mov_b32 m0, s2", "s_nop 0", LOAD, "v_readfirstlane_b32 s5, v0", ("s_cbranch_scc1 65531", 0), "s_endpgm"], 1),
    (["s_mov_b32 m0, s2", "s_nop 0", LOAD, "v_readfirstlane_b32 s5, v0", "s_nop 1", ("s_cbranch_scc1 65530", 0), "s_endpgm"], 0),
    # past a branch that is always taken
    (["v_readfirstlane_b32 s5, v0", ("s_branch 1", 3), "s_mov_b32 m0, s2", "s_nop 0", LOAD], 1),
    (["s_branch 1", "v_readfirstlane_b32 s5, v0", "s_endpgm", "s_mov_b32 m0, s2", "s_nop 0", LOAD], 0)])
def test_what_is_found(lines, bad):
    assert len(hazards(functions(listing_of(lines))["f"])) == bad


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{name: code} of the library's functions that load to LDS by assembly."""
    if not os.path.exists(hip_build.LIB):
        hip_build.build()
    here = tmp_path_factory.mktemp("isa")
    lib = shutil.copy(hip_build.LIB, here)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True)
    out = {}
    for name in sorted(os.listdir(here)):
        if "amdgcn" not in name:
            continue
        with open(here / name, "rb") as f:
            if not re.search(rb"(mv|ring|wide)_kernelI?\w*st2f86MmArgs", f.read()):
                continue
        r = subprocess.run([OBJDUMP, "-d", here / name], check=True, capture_output=True, text=True)
        out.update(functions(r.stdout))
    return {n: c for n, c in out.items() if any(i.to_lds for i in c)}


def test_the_library(kernels):
    for kind in ("mv_kernel", "ring_kernel", "wide_kernel"):
        assert any(kind in name for name in kernels), kind
    for name, code in kernels.items():
        assert not hazards(code), (name, sorted(hazards(code))[:5])
