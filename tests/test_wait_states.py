"""The waits that the machine leaves to the code, in the code objects of this build, checked on the CPU.

A vector memory instruction reads a scalar register (a buffer's descriptor, a base address) as a vector instruction
(v_readfirstlane, v_readlane of a spilled scalar, a compare) wrote it only five wait states later: an instruction is
one, s_nop n is n + 1. The compiler counts them for the instructions that it makes; to it an asm block is none,
so a load written in one has to bring its own."""
import glob
import os
import re
import subprocess

import pytest

from test_build_guard import BUILD, ROOT, _disassemble, _objects

STATES = 5
SDST_SECOND = re.compile(r"v_(add|sub|subrev|addc|subb|subbrev)_co|v_div_scale|v_mad_[ui]64")
TWO = re.compile(r"s\[(\d+):(\d+)\]$")


def scalars(operand):
    """The scalar registers that an operand names."""
    got = set()
    for word in operand.split():
        pair = TWO.match(word)
        if pair:
            got |= set(range(int(pair[1]), int(pair[2]) + 1))
        elif re.match(r"s\d+$", word):
            got.add(int(word[1:]))
    return got


def parse(text):
    """Instructions of a disassembly, function by function: (name, operands, address, jump or None)."""
    functions, here, base = [], [], 0
    for line in text.splitlines():
        head = re.match(r"([0-9a-f]+) <(.*)>:", line)
        if head:
            here, base = [], int(head[1], 16)
            functions.append((head[2], here))
            continue
        if "//" not in line:
            continue
        code, _, note = line.partition("//")
        name, _, rest = code.strip().partition(" ")
        to = re.search(r"<[^>+]*(?:\+0x([0-9a-f]+))?>", note) if name.startswith(("s_branch", "s_cbranch")) else None
        here.append((name, [x.strip() for x in re.split(r",", rest)], int(note.split(":")[0], 16), None if to is None else base + int(to[1] or "0", 16)))
    return functions


def short(function):
    """The vector memory instructions that may come too early, with the instruction before them."""
    at = {address: i for i, (_, _, address, _) in enumerate(function)}
    jumps = {}
    for i, (_, _, _, to) in enumerate(function):
        if to is not None:
            jumps.setdefault(at[to], []).append(i)

    def before(i):
        if i > 0 and not function[i - 1][0].startswith(("s_branch", "s_endpgm", "s_setpc")):
            yield i - 1
        yield from jumps.get(i, ())

    found = []
    for i, (name, operands, _, _) in enumerate(function):
        if not name.startswith(("buffer_", "global_", "scratch_", "flat_")):
            continue
        reads = set().union(*map(scalars, operands))
        todo, seen = [(j, 0) for j in before(i)] if reads else [], {}
        while todo:
            j, states = todo.pop()
            if states >= STATES or seen.get(j, STATES) <= states:
                continue
            seen[j] = states
            op, args, _, _ = function[j]
            writes = set()
            if op.startswith("v_"):
                writes = scalars(args[0]) | (scalars(args[1]) if SDST_SECOND.match(op) and len(args) > 1 else set())
            if writes & reads:
                found.append((name, operands, op, args, states))
                break
            states += int(args[0], 0) + 1 if op == "s_nop" else 1
            todo += [(k, states) for k in before(j)]
    return found


LISTING = """
0000000000001000 <one>:
	v_readlane_b32 s2, v9, 62          // 000000001000: 00000000
	s_add_u32 m0, s4, 0x1000           // 000000001008: 00000000
	s_nop {nop}                        // 000000001010: 00000000
	buffer_load_dwordx4 v1, s[0:3], 0 offen lds // 000000001014: 00000000
	s_cbranch_scc1 65530               // 00000000101C: 00000000 <one+0x8>
	v_cmp_lt_u32_e64 s[2:3], v0, v1    // 000000001020: 00000000
	s_branch 65530                     // 000000001028: 00000000 <one+0x14>
"""


@pytest.mark.parametrize("nop,loads", [(0, 2), (3, 1), (15, 1)])
def test_the_count(nop, loads):
    """Two ways to the load: straight on, and by the jump, behind which nothing is waited for."""
    (name, function), = parse(LISTING.format(nop=nop))
    assert name == "one" and len(function) == 7
    straight = [x for x in function if x[0] != "s_branch"]
    assert bool(short(straight)) == (nop < 3)
    assert len(short(function)) == 1
    assert len(short(function)) + len(short(straight)) == loads


@pytest.mark.parametrize("obj", sorted(os.path.basename(o) for o in glob.glob(os.path.join(BUILD, "*.o"))) or ["(none)"])
def test_descriptors_are_waited_for(obj, tmp_path):
    path, = [o for o in _objects() if os.path.basename(o) == obj]
    loads = 0
    for name, function in parse(_disassemble(path, tmp_path)):
        loads += sum(x[0].startswith(("buffer_load", "global_load", "global_store")) for x in function)
        found = short(function)
        assert not found, f"{name}: {len(found)} too early, e.g. {found[0]}"
    assert loads or obj == "bchip.o"


OFFSETS = """
#include "paged.hpp"
namespace bchip {
__global__ void probe(pg_u32x4 from, const uint8_t* at, uint32_t n, float* out) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[4096];
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, (int)n, 0x00020000);
    pg_lds* to = (pg_lds*)lds + 2048;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to, 4, 4 * threadIdx.x, 0, 0, 0);
    load_lds(from, 16 * threadIdx.x, (uint32_t)(uintptr_t)(pg_lds*)lds, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to, 4, 4 * threadIdx.x, 4096, 0, 0);
    __syncthreads();
    out[threadIdx.x] = ((float*)lds)[threadIdx.x];
}
}
"""


def test_the_compiler_sets_its_own_offsets_again(tmp_path):
    """Loads into LDS take their place from M0: one that the compiler makes behind load_lds, which sets it, does not
    find its own there any more. (Compiled, not run.)"""
    source, listing = tmp_path / "probe.hip", tmp_path / "probe.s"
    source.write_text(OFFSETS)
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "--cuda-device-only", "-S", "-O3", "-std=c++17", "-w", "-Xclang", "-target-feature",
                    "-Xclang", "-packed-fp32-ops", f"-I{ROOT}/include", f"-I{ROOT}/borrowed-compute_amd/csrc", str(source), "-o", str(listing)],
                   check=True, capture_output=True)
    steps = re.findall(r"^\s+(s_\w+ m0|buffer_load_\w+).*", listing.read_text(), re.M)
    assert [x.split("_")[0] for x in steps] == ["s", "buffer"] * 3, steps
