"""The full tile of the 8-bit products (fp8_gemm.hip) and the weight gradients (fp8_grad.hip) issue their matrix instructions and
their DMA to LDS as inline assembly, so the compiler inserts none of the wait states that matrix instructions need. This checks on
the compiler's own gfx950 assembly, for every kernel of the two:

- a register that a matrix instruction reads (an operand or its scales) was not written by a vector instruction in the wait states
  before it, on any path that the control flow allows (a fixed point over the basic blocks, loops included);
- no instruction but a matrix instruction reads an accumulator within 32 wait states of one, on any path;
- accumulators are not moved inside the walk, and nothing spills."""
import re
import subprocess
import tempfile
from pathlib import Path

import pytest

from nanochat_amd import native
from tests.test_prefill_gemm_isa import blocks, loop_lines, regs, wait_states_before_agpr_reads, writer_kind

ASM = {"gemm": ("fp8_gemm.hip", r"_ZN2nc12_GLOBAL__N_115fp8_gemm_kernelINS0_6FgTileILi8ELi2ELi2ELi2EEELi([012])EEEvNS0_6F8GemmEi"),
       "grad": ("fp8_grad.hip", r"_ZN2nc12_GLOBAL__N_115fp8_grad_kernelILi([0123])EEEvNS0_7F8GradsE")}
KERNELS = [("gemm", e) for e in range(3)] + [("grad", m) for m in range(4)]


@pytest.fixture(scope="module")
def kernels():
    bodies, texts = {}, []
    for name, (source, symbol) in ASM.items():
        with tempfile.TemporaryDirectory() as tmp:
            out = Path(tmp) / "k.s"
            subprocess.run([native.hipcc(), *native.HIPCC_FLAGS, f"-I{native.CSRC}", "--cuda-device-only", "-S", "-o", str(out),
                            str(native.CSRC / source)], check=True, capture_output=True)
            texts.append(out.read_text())
        for m in re.finditer(rf"^({symbol}):[^\n]*\n(.*?)\n\.Lfunc_end", texts[-1], re.S | re.M):
            bodies[(name, int(m.group(2)))] = m.group(3).splitlines()
    return bodies, texts


def operands(ops):
    """The vector registers a matrix instruction reads beside its accumulator: both operands, and scales where it has them."""
    return set().union(*(regs(t.split()[0]) for t in ops[1:3] + ops[4:6] if t))


def least_wait_states(lines, far=1 << 20):
    """The fewest wait states between a vector instruction that writes a register and a matrix instruction that reads it as an
    operand, over every path (s_nop N counts N + 1, any other instruction 1; a later write by an LDS read replaces the first)."""
    bl = blocks(lines)
    index = {lab: i for i, (lab, _, _) in enumerate(bl)}
    state_in, work, fewest = {0: {}}, [0], far
    while work:
        i = work.pop()
        age = dict(state_in[i])   # register -> wait states since a vector instruction wrote it
        for mn, ops in bl[i][1]:
            if mn.startswith("v_mfma"):
                fewest = min([fewest] + [age[r] for r in operands(ops) if r in age])
            kind = writer_kind(mn, ops)
            step = int(ops[0], 0) + 1 if mn == "s_nop" else 1
            age = {r: a + step for r, a in age.items() if a + step < 64}
            if kind:
                for r in regs(ops[0]):
                    age.pop(r, None)
                    if kind == "valu":
                        age[r] = 0
        for t in bl[i][2]:
            k = index[t]
            old = state_in.get(k)
            new = age if old is None else {r: min(old.get(r, far), age.get(r, far)) for r in old.keys() | age.keys()}
            if new != old:
                state_in[k] = new
                work.append(k)
    return fewest


def test_every_kernel_is_built(kernels):
    bodies, texts = kernels
    assert sorted(bodies) == sorted(KERNELS)
    for b in bodies.values():
        assert not any("scratch_" in line for line in b)
    for text in texts:
        counts = re.findall(r"\.[sv]gpr_spill_count:\s+(\d+)", text)
        assert counts and all(int(c) == 0 for c in counts)


@pytest.mark.parametrize("epi,wide,narrow", [(0, 32, 0), (1, 16, 8)])
def test_a_tiles_stores_are_as_many_as_its_successor_counts(kernels, epi, wide, narrow):
    """The wait for a tile's first stage lets that many newer stores of the last tile's be on their way."""
    count = lambda mn: sum(line.strip().startswith(mn) for line in kernels[0][("gemm", epi)])   # noqa: E731
    assert count("buffer_store_dwordx4") == wide and count("buffer_store_byte") == narrow
    assert count("global_store") == count("flat_store") == 0


@pytest.mark.parametrize("which", KERNELS)
def test_operands_are_not_written_right_before(kernels, which):
    # 2 are needed; both kernels read their operands a phase or a stage ahead
    assert sum("v_mfma" in line for line in kernels[0][which]) >= 32
    assert least_wait_states(kernels[0][which]) >= 2


@pytest.mark.parametrize("which", KERNELS)
def test_accumulators_stay_in_place(kernels, which):
    walk = [body for _, body, _ in blocks(kernels[0][which]) if any(mn.startswith("v_mfma") for mn, _ in body)]
    assert walk and any("v_mfma" in line for line in loop_lines(kernels[0][which]))
    for body in walk:   # what a tile's results read stands behind the last product, in a block of its own or at the end of one
        last = max(i for i, (mn, _) in enumerate(body) if mn.startswith("v_mfma"))
        assert not [i for i, (mn, _) in enumerate(body) if mn.startswith("v_accvgpr") and i < last and mn != "v_accvgpr_write_b32"]


@pytest.mark.parametrize("which", KERNELS)
def test_accumulators_read_after_the_wait_states(kernels, which):
    assert wait_states_before_agpr_reads(kernels[0][which]) >= 32


def test_the_check_sees_a_write_right_before():
    loop = """
        ds_read_b128 v[0:3], v20
.LBB0_1:                                ; =>This Inner Loop Header: Depth=1
        v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[0:7], v[8:15], a[0:3], v30, v31 op_sel_hi:[0,0,0]
        v_lshrrev_b32_e32 v30, 8, v30
        s_nop 4
        s_cbranch_scc1 .LBB0_1
; %bb.2:
        s_endpgm""".splitlines()
    assert least_wait_states(loop) == 6
    assert least_wait_states([line.replace("v30, 8, v30", "v40, 8, v40") for line in loop]) == 1 << 20
