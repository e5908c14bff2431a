"""The waits of the MXFP4 GEMM (kadan_amd/csrc/mxfp4_dense.hip), read from the built library.

gemm_kernel's rows of x pass through LDS: every wavefront copies a share of each chunk, three
chunks ahead, and reads what the others copied once all are past a barrier.  A wavefront's
memory operations return in order and it waits for "all but the last N of them", so N may not
exceed what was issued behind the copies that the barrier stands for, in the loop's first turn
as in all later ones.  A wait for too few shows on the device only when wavefronts drift apart;
here the compiled instructions are followed through three turns of the loop, counting."""
import os
import re
import shutil
import subprocess

import pytest

import kadan_amd

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
LIBRARY = os.path.join(os.path.dirname(kadan_amd.__file__), "libkadan_amd.so")
KERNEL = re.compile(r"<_ZN\w*11gemm_kernelILi(\d)ELb(\d)ELi(\d)ELi(\d)EEEvNS0_4GemmE>:")
BARRIERS = 12  # three turns of four chunks


def code(folder):
    """{(TT, SPLIT, OPS, OUT): [(address, instruction)]} of every gemm_kernel of the library."""
    copy = shutil.copy(LIBRARY, folder)
    subprocess.run([OBJDUMP, "--offloading", copy], cwd=folder, check=True, capture_output=True)
    kernels = {}
    for name in sorted(os.listdir(folder)):
        if "gfx950" not in name:
            continue
        path = os.path.join(folder, name)
        if b"4GemmE" not in open(path, "rb").read():
            continue
        text = subprocess.run([OBJDUMP, "-d", path], check=True, capture_output=True,
                              text=True).stdout
        body = None
        for line in text.splitlines():
            if line.endswith(">:"):
                match = KERNEL.search(line)
                body = kernels.setdefault(tuple(map(int, match.groups())), []) if match else None
            elif body is not None and "//" in line:
                instruction, at = line.split("//", 1)
                body.append((int(at.split(":")[0], 16), instruction.strip()))
    return kernels


def run(body):
    """The memory operations outstanding at each of the first barriers: (which of the copies to
    LDS are still on their way as ("x" | "scale", number from 0), reads of LDS on their way)."""
    place = {at: i for i, (at, _) in enumerate(body)}
    flying, reads, issued, barriers, i = [], 0, {"x": 0, "scale": 0}, [], 0
    while len(barriers) < BARRIERS:
        at, text = body[i]
        op, i = text.split()[0], i + 1
        if op.startswith(("buffer_", "global_", "flat_", "scratch_")):
            kind = None
            if text.endswith(" lds"):
                kind = "x" if op.endswith("x4") else "scale"
            flying.append((kind, issued.get(kind)))
            if kind:
                issued[kind] += 1
        elif op.startswith("ds_"):
            reads += 1
        elif op == "s_waitcnt":
            left = re.search(r"vmcnt\((\d+)\)", text)
            if left and int(left[1]) < len(flying):
                flying = flying[len(flying) - int(left[1]):]
            left = re.search(r"lgkmcnt\((\d+)\)", text)
            if left:
                reads = min(reads, int(left[1]))
        elif op == "s_barrier":
            barriers.append(([f for f in flying if f[0]], reads))
        elif op.startswith(("s_branch", "s_cbranch")):
            # (the loop's own way: back every time; conditional jumps ahead leave it, or skip
            # what a chunk past the end has no use for)
            step = int(text.split()[1])
            target = place[at + 4 + 4 * (step - 65536 if step >= 32768 else step)]
            if op == "s_branch" or target < i:
                i = target
        assert op != "s_endpgm", "the loop ended before it began"
    return barriers, issued


def test_every_barrier_stands_for_its_chunks_copies(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    kernels = code(str(tmp_path))
    assert {k[2] for k in kernels} == {0, 1, 2} and {k[0] for k in kernels} == {1, 2, 3, 4}
    for (tiles, split, operands, out), body in sorted(kernels.items()):
        name = f"gemm_kernel<{tiles}, {split}, {operands}, {out}>"
        barriers, issued = run(body)
        copies = -(-(2 * tiles * 32 * 40 // 256) // 8) if operands == 1 else 0  # of four chunks
        assert issued["x"] == (BARRIERS + 2) * tiles, name
        for chunk, (flying, reads) in enumerate(barriers):
            arrived = {"x": (chunk + 1) * tiles, "scale": (chunk // 4 + 1) * copies}
            late = [f for f in flying if f[1] < arrived[f[0]]]
            assert not late, f"{name}: chunk {chunk} is read while {late} may not be there"
            assert not reads, f"{name}: chunk {chunk}'s buffers are written while they are read"
