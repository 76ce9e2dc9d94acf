"""All but the full tiles of the 8-bit products (fp8_gemm.hip: wide, half and small ones; fp8_skinny.hip: fp8_some_kernel) read stages from LDS
that DMA issued as inline assembly brings, and wait for them by a number of newer memory instructions: that number has to be on
its way behind a stage's DMA on every path, or a wait for it lets the stage itself be late. What the compiler moves of its own loads and
stores could change it. This checks on the compiler's gfx950 assembly, for every such kernel:

- at each barrier of the walk, the stage read behind it has landed on every path that the control flow allows: its DMA are waited for
  by an s_waitcnt whose vmcnt is at most the number of memory instructions issued since (a fixed point over the basic blocks);
- this wave's own LDS reads are done at each of them: the DMA behind it fills the slot that they read;
- no DMA is on its way where a kernel ends."""
import re
import subprocess
import tempfile
from pathlib import Path

import pytest

from nanochat_amd import native
from tests.test_prefill_gemm_isa import blocks

# stages in LDS, 16-byte DMA of a stage and wave
KERNELS = {("fp8_gemm.hip", f"15fp8_gemm_kernelINS0_6FgTileI{tile}EELi{epi}EEEv"): sizes
           for tile, sizes in (("Li2ELi1ELi4ELi2E", (2, 8)), ("Li1ELi1ELi4ELi3E", (3, 6))) for epi in range(3)}
KERNELS |= {("fp8_gemm.hip", f"15fp8_gemm_kernelINS0_6FgTileI{tile}EELi3EEEv"): (2, 8)   # exact products before a ReLU^2
            for tile in ("Li2ELi1ELi4ELi2E", "Li4ELi2ELi4ELi2E")}
KERNELS |= {("fp8_skinny.hip", "15fp8_some_kernelILi1ELi8EEEv"): (3, 4), ("fp8_skinny.hip", "15fp8_some_kernelILi2ELi4EEEv"): (4, 2)}
LANDED = 1 << 20
VMEM = ("buffer_", "global_", "flat_", "scratch_")


@pytest.fixture(scope="module")
def bodies():
    out = {}
    for source in sorted({s for s, _ in KERNELS}):
        with tempfile.TemporaryDirectory() as tmp:
            asm = Path(tmp) / "k.s"
            subprocess.run([native.hipcc(), *native.HIPCC_FLAGS, f"-I{native.CSRC}", "--cuda-device-only", "-S", "-o", str(asm),
                            str(native.CSRC / source)], check=True, capture_output=True)
            text = asm.read_text()
        for _, name in (k for k in KERNELS if k[0] == source):
            m, = re.finditer(rf"^_ZN2nc12_GLOBAL__N_1{name}\w*:[^\n]*\n(.*?)\n\.Lfunc_end", text, re.S | re.M)
            out[(source, name)] = m.group(1).splitlines()
    return out


def counter(ops, name):
    """The count that an s_waitcnt waits for, or None."""
    m = re.search(rf"{name}\((\d+)\)", " ".join(ops))
    return int(m.group(1)) if m else None


def in_a_loop(bl):
    """The blocks that some path from them leads back to."""
    index = {lab: i for i, (lab, _, _) in enumerate(bl)}
    succ = [[index[t] for t in s] for _, _, s in bl]

    def reach(i):
        seen, work = set(), list(succ[i])
        while work:
            k = work.pop()
            if k not in seen:
                seen.add(k)
                work.extend(succ[k])
        return seen
    return {i for i in range(len(bl)) if i in reach(i)}


def faults(lines, ring, loads):
    """(barriers of the walk, what is wrong at them and at the ends). A state: for the last `ring` stages' DMA, newest first, the
    fewest memory instructions issued since, LANDED once waited for; and whether LDS reads may be outstanding. States are kept apart
    by the walk's last barrier: its steps follow one another in the listing's order and it ends with the first that is left out,
    which the branches do not show, so paths that leave one out and go on are not followed."""
    bl = blocks(lines)
    index = {lab: i for i, (lab, _, _) in enumerate(bl)}
    looped = in_a_loop(bl)
    steps = [(i, at) for i in sorted(looped) for at, (mn, _) in enumerate(bl[i][1]) if mn == "s_barrier"]
    start = (0, len(steps) - 1)
    state_in, work, wrong = {start: ((LANDED,) * ring * loads, LANDED, False)}, [start], {}
    while work:
        i, step = node = work.pop()
        ages, small, reading = state_in[node]   # small: of the oldest 4-byte DMA that has not landed
        for at, (mn, ops) in enumerate(bl[i][1]):
            if mn.startswith(VMEM):
                ages, small = tuple(min(a + 1, LANDED) for a in ages), min(small + 1, LANDED)
                if "lds" in " ".join(ops).split():
                    if "dwordx4" in mn:
                        ages = (0,) + ages[:-1]
                    else:
                        small = min(small, 0)
            elif mn.startswith("ds_read"):
                reading = True
            elif mn == "s_waitcnt":
                n, k = counter(ops, "vmcnt"), counter(ops, "lgkmcnt")
                if n is not None:
                    ages, small = tuple(LANDED if a >= n else a for a in ages), LANDED if small >= n else small
                reading = reading and k != 0
            elif (i, at) in steps:
                step = (step + 1) % len(steps)
                if steps[step] != (i, at):
                    break
                # on their way may be the ring - 2 stages behind the one that is read
                wrong[(i, at)] = [f"stage late by {a}" for a in ages[(ring - 2) * loads:(ring - 1) * loads] if a != LANDED] + \
                    ["LDS reads"] * reading
            elif mn == "s_endpgm":
                wrong[(i, at)] = ["DMA at the end"] * (any(a != LANDED for a in ages) or small != LANDED)
        else:
            for t in bl[i][2]:
                k, new = (index[t], step), (ages, small, reading)
                old = state_in.get(k)
                if old is not None:
                    new = (tuple(map(min, old[0], ages)), min(old[1], small), old[2] or reading)
                if new != old:
                    state_in[k] = new
                    work.append(k)
    return sum(at in wrong for at in steps), [(bl[i][0], what) for (i, _), found in sorted(wrong.items()) for what in found]


@pytest.mark.parametrize("which", KERNELS, ids=lambda k: k[1])
def test_a_stage_has_landed_where_it_is_read(bodies, which):
    barriers, wrong = faults(bodies[which], *KERNELS[which])
    assert barriers >= 4 and not wrong, wrong


@pytest.mark.parametrize("which", KERNELS, ids=lambda k: k[1])
def test_the_check_sees_a_wait_that_lets_one_more_be_late(bodies, which):
    """In the listing: every wait for memory in front of a step's barrier lets as many more be on their way as its slack is, and one
    more: none, but for the two loads that fp8_some_kernel leaves to the compiler."""
    ring, loads = KERNELS[which]
    more = 3 if "some" in which[1] else 1
    raised = [re.sub(r"vmcnt\((\d+)\)", lambda m: f"vmcnt({int(m.group(1)) + more})", line) for line in bodies[which]]
    assert faults(raised, ring, loads)[1]
