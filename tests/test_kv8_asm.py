"""The 8-bit cache's kernels as compiled (CPU only: compiles k_kv8.hip for gfx950
and reads the assembly).

k_kv8_attn_rows stages K and V by DMA into LDS, six instructions of a wave in each
phase, and waits for the ones two phases back by count: vmcnt(9) before a
phase's barrier, vmcnt(12) where the last block's V is cleared. That holds only if the
loop issues nothing else to the queue. No kernel of the file may use accumulator
registers: the compiler restores values from them before the lane mask where lanes
have diverged."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "enginesmith-qwen35-08b-long-decode-m5max-round005_amd")
HIPCC = "/opt/rocm/bin/hipcc"
VMEM = re.compile(r"(global|buffer|flat|scratch)_(load|store|atomic)")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    if not os.path.exists(HIPCC) or shutil.which("ld.lld", path="/opt/rocm/llvm/bin") is None:
        pytest.skip("hipcc for gfx950 is not installed")
    out = tmp_path_factory.getbasetemp() / "k_kv8.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fhip-fp32-correctly-rounded-divide-sqrt",
                    "-ffp-contract=off", "-I" + os.path.join(ROOT, "include"), "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "--cuda-device-only", "-S", "-o", str(out),
                    os.path.join(PKG, "csrc", "k_kv8.hip")], check=True, capture_output=True, cwd=os.path.join(PKG, "csrc"))
    return [l.split(";")[0].strip() if not l.strip().startswith(".LBB") else l.strip() for l in out.read_text().splitlines()]


def test_no_accumulator_registers(asm):
    assert not [l for l in asm if "accvgpr" in l or re.search(r"\ba\[?\d", l)]


def test_the_loop_of_many_rows_counts_its_loads(asm):
    start = next(i for i, l in enumerate(asm) if re.match(r"_ZN2es12_GLOBAL__N_1\d+k_kv8_attn_rows\w*:", l))
    body = asm[start:next(i for i in range(start, len(asm)) if asm[i] == "s_endpgm")]
    head = next(i for i, l in enumerate(body) if "Loop Header" in l)
    label = body[head].split(":")[0]
    # the loop's blocks, wherever they stand
    marks = [i for i, l in enumerate(body) if l.startswith(".LBB")] + [len(body)]
    loop = [l for i, j in zip(marks, marks[1:]) if i == head or f"Header=BB{label[4:]} " in body[i] for l in body[i:j]]
    assert sum(l.startswith("v_mfma_scale_f32_32x32x64") for l in loop) == 32, "scores and values of one block"
    vmem = [l for l in loop if VMEM.match(l)]
    assert len(vmem) == 12 and all(l.endswith(" lds") for l in vmem), vmem
    waits = [int(m.group(1)) for l in loop if (m := re.search(r"vmcnt\((\d+)\)", l))]
    assert sorted(waits) == [9, 9, 12, 12], waits
    barriers = [i for i, l in enumerate(loop) if l == "s_barrier"]
    assert len(barriers) == 2
