"""The order of DMA, waits and barriers in k_kv8_attn_rows, replayed on the CPU
from the kernel as compiled: whatever a half of the waves reads from LDS has
been waited for by every wave, and published by a barrier, before the read."""
import re

import pytest

from test_kv8_asm import asm  # noqa: F401  (the fixture)

GROUP = 6  # DMA instructions of a wave for one block: K, K, K's power, V, V, V's power


def steps(asm):
    """DMA instructions, waits for them, barriers, labels and branches, in the order of the text."""
    start = next(i for i, l in enumerate(asm) if re.match(r"_ZN2es12_GLOBAL__N_1\d+k_kv8_attn_rows\w*:", l))
    out = []
    for l in asm[start + 1:]:
        if l == "s_endpgm":
            return out
        if l.startswith(".LBB") or l.startswith("s_cbranch") or l.startswith("s_branch"):
            out.append(("edge", l))
        elif l == "s_barrier":
            out.append(("barrier", 0))
        elif re.match(r"buffer_load\w* .* lds$", l):
            out.append(("dma", 0))
        elif l.startswith("s_waitcnt") and (m := re.search(r"vmcnt\((\d+)\)", l)):
            out.append(("wait", int(m.group(1))))
    raise AssertionError("no end")


def waited(kinds, at):
    """vmcnt of the wait in front of the barrier `at`, in its own stretch of code; None if there is none."""
    for kind, n in reversed(kinds[:at]):
        if kind == "wait":
            return n
        if kind != "barrier" and kind != "dma":
            return None
    return None


@pytest.fixture(scope="module")
def counts(asm):  # noqa: F811
    """Waits in front of a phase's barrier and of the one that ends the half without the last block."""
    kinds = steps(asm)
    dma = [i for i, (kind, _) in enumerate(kinds) if kind == "dma"]
    barriers = [i for i, (kind, _) in enumerate(kinds) if kind == "barrier"]
    first = next(i for i in barriers if i > dma[0])
    ahead = sum(i < first for i in dma)
    phases = {waited(kinds, i) for i in barriers if first < i < dma[-1]}
    closing = next(i for i in barriers if i > dma[-1])
    assert len(phases) == 1, phases
    return ahead, phases.pop(), waited(kinds, closing)


class Half:
    """One half's waves: what they have issued and, at least, received; barriers passed so far."""

    def __init__(self, ahead):
        self.issued = [("kv"[i % GROUP // 3], i // GROUP) for i in range(ahead)]
        self.have, self.at_barrier, self.reads = 0, [], []

    def wait(self, n):
        if n is not None:
            self.have = max(self.have, len(self.issued) - n)

    def barrier(self):
        self.at_barrier.append(self.have)

    def read(self, what, block):
        self.reads.append((what, block, len(self.at_barrier)))


def replay(blocks, ahead, phase_wait, closing_wait):
    halves = [Half(ahead), Half(ahead)]
    for upper, half in enumerate(halves):
        def phase(p):
            half.wait(phase_wait)
            half.barrier()
            half.issued += [("k", p + 2)] * 3 + [("v", p + 2)] * 3
        if upper:
            phase(0)
        for b in range(upper, blocks, 2):
            phase(b)
            half.read("k", b)
            phase(b + 1)
            half.read("v", b)
        if blocks % 2 == upper:
            half.wait(closing_wait)
            half.barrier()
    return halves


def unsafe(blocks, *counts):
    """Reads of bytes that some half's waves may still be waiting for."""
    halves = replay(blocks, *counts)
    assert len(halves[0].at_barrier) == len(halves[1].at_barrier), "a barrier that one half never reaches"
    bad = []
    for half in halves:
        for what, block, barriers in half.reads:
            for other in halves:
                have = other.at_barrier[barriers - 1]
                need = max(i for i, x in enumerate(other.issued) if x == (what, block)) + 1
                if have < need:
                    bad.append((what, block))
    return bad


@pytest.mark.parametrize("blocks", [1, 2, 3, 4, 5, 8, 9, 64, 511])
def test_every_read_is_waited_for(counts, blocks):
    assert unsafe(blocks, *counts) == []


def test_the_replay_sees_a_missing_wait():
    for blocks in range(1, 7):
        assert ("v", blocks - 1) in unsafe(blocks, 2 * GROUP, 9, None)
        assert unsafe(blocks, 2 * GROUP, 9, 12) == []
        assert unsafe(blocks, 2 * GROUP, 9, 13) != []
        assert unsafe(blocks, 2 * GROUP, 10, 12) != []
