"""The MFMAs of the 4-bit GEMM tiles (gemm_mxfp4.hip) are inline asm, hidden from the
compiler's hazard recognizer.  This CPU test compiles the file for gfx950 to assembly and
checks, for every tile kernel:
  - nothing but MFMAs reads or writes an accumulator within 18 wait states behind an MFMA
    (as test_isa_mfma_acc.py, whose walk it uses);
  - neither of the two instructions before an MFMA writes one of its scale registers, which
    permutes write;
  - no register is spilled to memory: a spill would count among the copies that are waited for.
The kernel of several rounds counts on its stores: a tile's first step waits until at most
32 accesses are under way, the stores behind its copies, so at least as many stores of 16
bytes must be there, and no other access to memory but the copies."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from test_isa_mfma_acc import CSRC, WAIT_STATES, _check, _is_insn, _regs

TILES = 12  # kernels: 256 (plain, staged, edge, rounds), 128 (2 or 3 stages, whole, tail)


def _scale_writes(body):
    """MFMAs of whose scale registers one of the two instructions before writes one."""
    insns = [l for l in body if _is_insn(l)]
    bad = 0
    for i, line in enumerate(insns):
        if not line.startswith("v_mfma_scale"):
            continue
        scales = set()
        for operand in re.sub(r"^\S+\s+", "", line).split(",")[4:6]:
            scales |= _regs(operand.split()[0])
        for before in insns[max(0, i - 2):i]:
            if before.startswith(("v_", "ds_read")) and not before.startswith("v_mfma"):
                bad += bool(_regs(before.split(",")[0]) & scales)
    return bad


def _in_order(body):
    """The instructions, or where the sums are read ahead of the MFMAs (the kernel of several
    rounds, whose loop the compiler turned): the block that reads them behind an MFMA, which
    any way into it may have as its last."""
    mfma = next(i for i, l in enumerate(body) if l.startswith("v_mfma"))
    read = next(i for i, l in enumerate(body) if l.startswith("v_accvgpr_read"))
    if read > mfma:
        return body
    label = max(i for i in range(read) if body[i].endswith(":"))
    return [body[mfma]] + body[label:mfma]


@pytest.fixture(scope="module")
def bodies(tmp_path_factory):
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc) or shutil.which("python3") is None:
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("isa") / "mxfp4.s"
    subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", "-munsafe-fp-atomics",
                    "--cuda-device-only", "-S", "-I" + os.path.join(CSRC, "_build"),
                    os.path.join(CSRC, "gemm_mxfp4.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    found = re.findall(r"^(_Z\S*gemm_mxfp4(?:_128|_rounds)?_kernel\S*):[^\n]*\n(.*?)^\.Lfunc_end",
                       out.read_text(), re.S | re.M)
    return {name: [l.split(";")[0].strip() for l in body.split("\n")] for name, body in found}


def test_accumulators_and_scales(bodies):
    assert len(bodies) == TILES, sorted(bodies)
    for name, body in bodies.items():
        mfmas = [l for l in body if l.startswith("v_mfma")]
        assert len(mfmas) >= 64 and {l.split()[0] for l in mfmas} == {
            "v_mfma_scale_f32_16x16x128_f8f6f4"}, name
        assert all(l.split()[1].startswith("a[") for l in mfmas), name
        walk = _in_order(body)
        assert WAIT_STATES <= _check(walk)[2] < 10 ** 9, name
        assert _check(body)[2] >= WAIT_STATES, name
        assert _scale_writes(body) == 0, name
        assert not any(l.startswith("scratch_") for l in body), name
        # the checks fire: an early read of a sum, and a permute moved before its use
        last = max(i for i, l in enumerate(walk) if l.startswith("v_mfma"))
        early = walk[:last + 1] + ["v_accvgpr_read_b32 v0, a0"] + walk[last + 1:]
        assert _check(early)[2] < WAIT_STATES, name
        at = next(i for i, l in enumerate(body) if l.startswith("v_mfma"))
        scale = body[at].split(",")[4].split()[0]
        assert _scale_writes(body[:at] + [f"v_perm_b32 {scale}, v0, v1, v2"] + body[at:]) > 0


def test_stores_of_rounds(bodies):
    (body,) = [b for n, b in bodies.items() if "rounds" in n]
    waits = [l for l in body if re.match(r"s_waitcnt vmcnt\((?!0\))", l)]
    assert waits and set(waits) == {"s_waitcnt vmcnt(32) lgkmcnt(0)"}
    memory = [l for l in body if re.match(r"(global|flat|buffer|scratch)_", l)]
    stores = [l for l in memory if not re.match(r"buffer_load_dwordx4 .*\blds$", l)]
    assert len(stores) >= 32 and {l.split()[0] for l in stores} == {"global_store_dwordx4"}
    # behind the last MFMA of a tile, and no copy among them
    order = [l for l in body if l.startswith(("v_mfma", "buffer_load", "global_store"))]
    first = next(i for i, l in enumerate(order) if l.startswith("global_store"))
    assert all(l.startswith("global_store") for l in order[first:first + len(stores)])
