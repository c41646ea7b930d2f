"""The attention of a tree of drafted tokens as compiled (CPU only: compiles k_tree.hip
for gfx950 and reads the assembly).

k_tree_attn stages K and V by DMA into LDS, four instructions of a wave in each step of
32 keys, and waits by count for those of the step at hand: vmcnt(8) with two steps
behind it on their way, vmcnt(4) with one, vmcnt(0) with none. That holds only if the loop
issues nothing else to the queue. No kernel of the file may use accumulator
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
    out = tmp_path_factory.getbasetemp() / "k_tree.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fhip-fp32-correctly-rounded-divide-sqrt",
                    "-ffp-contract=off", "-I" + os.path.join(ROOT, "include"), "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "--cuda-device-only", "-S", "-o", str(out),
                    os.path.join(PKG, "csrc", "k_tree.hip")], check=True, capture_output=True, cwd=os.path.join(PKG, "csrc"))
    return [l.split(";")[0].strip() for l in out.read_text().splitlines()]


def test_no_accumulator_registers(asm):
    assert not [l for l in asm if "accvgpr" in l or re.search(r"[\s,]a(\d|\[)", l)]


def test_the_loop_counts_its_loads(asm):
    start = next(i for i, l in enumerate(asm) if re.match(r"_ZN2es12_GLOBAL__N_1\d+k_tree_attn\w*:", l))
    body = asm[start:next(i for i in range(start, len(asm)) if asm[i] == "s_endpgm")]
    labels = {l[:-1]: i for i, l in enumerate(body) if l.startswith(".LBB")}
    product = next(i for i, l in enumerate(body) if l.startswith("v_mfma_f32_32x32x16_bf16"))
    spans = []  # from a backward branch's target to the branch, around a product
    for i, l in enumerate(body):
        m = re.match(r"s_c?branch\w*\s+(\.LBB\w+)", l)
        if m and labels[m.group(1)] < product < i:
            spans.append((labels[m.group(1)], i))
    loop = body[min(a for a, _ in spans):max(b for _, b in spans) + 1]
    assert sum(l.startswith("v_mfma_f32_16x16x32_bf16") for l in loop) == 16, "scores of 16 keys and 32 queries"
    assert sum(l.startswith("v_mfma_f32_32x32x16_bf16") for l in loop) == 8, "values of 16 keys"
    vmem = [l for l in loop if VMEM.match(l)]
    assert len(vmem) == 4 and all(l.endswith(" lds") for l in vmem), vmem
    waits = [int(m.group(1)) for l in loop if (m := re.search(r"vmcnt\((\d+)\)", l))]
    assert sorted(waits) == [0, 4, 8], waits
    assert sum(l == "s_barrier" for l in loop) == 1
