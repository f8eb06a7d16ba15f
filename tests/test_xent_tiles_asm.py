"""CPU: the K loops of the cross entropy operator's tile kernels (csrc/xent_tiles.hip), checked in the compiler's output.

A step's counted wait, vmcnt(stages on their way behind the next one), holds only while the loop's vector-memory stream is
exactly the DMA instructions that the source issues: neither a register spilled into the loop nor any other access may join
it.  The DMA takes its LDS address from M0, which no other instruction of these kernels may write."""
import os
import re
import subprocess

import pytest

from test_kloop_asm import CSRC, HIPCC, ROOT, _is_dma, _kernel


def _k_loop(ins):
    """the shortest loop among those that hold the most MFMAs (around it there may be one over tiles)"""
    labels = {a: i for i, (op, a) in enumerate(ins) if op == "label"}
    loops = [ins[labels[a.strip()]:i + 1] for i, (op, a) in enumerate(ins)
             if (op.startswith("s_cbranch") or op == "s_branch") and labels.get(a.strip(), i) < i]
    return max(loops, key=lambda body: (sum(o.startswith("v_mfma") for o, _ in body), -len(body)))


@pytest.fixture(scope="module")
def text(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not present")
    out = tmp_path_factory.mktemp("xent") / "xent_tiles.s"
    subprocess.run([HIPCC, "-O3", "-std=c++17", "-fPIC", "--offload-arch=gfx950", "-I" + os.path.join(ROOT, "include"),
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-S", "--cuda-device-only",
                    os.path.join(CSRC, "xent_tiles.hip"), "-o", str(out)], check=True, capture_output=True)
    return open(out).read()


@pytest.mark.parametrize("wide", [0, 1])
@pytest.mark.parametrize("tile", [128, 256])
@pytest.mark.parametrize("pkc,qkc,logits", [(1, 1, 1), (0, 1, 0), (0, 0, 0)], ids=["logits", "dx", "dw"])
def test_k_loop(text, tile, pkc, qkc, logits, wide):
    name, ins = _kernel(text, f"_ZN10asl_detail16xent_tile_kernelILi{tile}ELb{pkc}ELb{qkc}ELb{logits}ELb{wide}EE")
    loop = _k_loop(ins)
    depth = 64 if pkc or qkc else 32
    stages, dma = 128 // depth, 2 * tile * depth // 2048                # DMA instructions a wave issues for a stage
    slices, frags = 128 // 16, tile // 64
    assert sum(o.startswith("v_mfma") for o, _ in loop) == slices * frags * frags
    assert sum(_is_dma(o, a) for o, a in loop) == stages * dma
    for op, a in loop:
        assert not op.startswith(("scratch_", "global_", "flat_")), f"{op} {a} inside the K loop"
        assert not op.startswith("buffer_") or _is_dma(op, a), f"{op} {a} inside the K loop"
    waits = [int(re.search(r"vmcnt\((\d+)\)", a).group(1)) for op, a in loop if op == "s_waitcnt" and "vmcnt" in a]
    assert waits == [(stages - 2) * dma] * stages
    assert sum(op == "s_barrier" for op, _ in loop) == stages
    # fragments: 16 bytes of a row contiguous along k, or two transposing reads of 8
    reads = {"ds_read_b128": (pkc + qkc) * slices * frags, "ds_read_b64_tr_b16": (2 - pkc - qkc) * 2 * slices * frags}
    for op, n in reads.items():
        assert sum(o == op for o, _ in loop) == n, op
    written = [a for _, a in ins if re.match(r"m0\b", a)]
    assert len(written) == sum(_is_dma(o, a) for o, a in ins), "M0 written by something else"


@pytest.mark.parametrize("wide", [0, 1])
def test_k_loops_of_the_pair(text, wide):
    _, ins = _kernel(text, f"_ZN10asl_detail21xent_tile_pair_kernelILi128ELb{wide}EE")
    assert not any(op.startswith("scratch_") for op, _ in ins)
    assert sum(bool(re.match(r"m0\b", a)) for _, a in ins) == sum(_is_dma(o, a) for o, a in ins)
