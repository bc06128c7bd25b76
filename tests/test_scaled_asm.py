"""Compiled code of the scaled operators' kernels whose MFMAs are inline assembly, which the compiler
schedules without knowing their hazards.

scaled_dma16_kernel: gemm_dma16_kernel's k loop in front of another epilogue. grad_dma_kernel: an MFMA may read a vector register no sooner than two instructions after an ordinary
vector instruction has written it; its accumulators are read only after the k loop, behind the wait
states the kernel puts there; and, as in gemm_dma_kernel, M0 belongs to the DMA sequences and nothing
in the k loop waits for vector memory but the kernel's own waits."""
import re

import pytest

from test_dma_asm import asm, kernel_body  # noqa: F401  (the fixture compiles the sources once)


def names(text, kernel):
    return sorted(set(re.findall(r"^(_Z\S*%s\S*):" % kernel, text, flags=re.M)))


def registers(operand):
    """The numbers of a vector register operand ("v7", "v[8:11]"; AGPRs are none)."""
    m = re.fullmatch(r"v(\d+)", operand)
    if m:
        return {int(m.group(1))}
    m = re.fullmatch(r"v\[(\d+):(\d+)\]", operand)
    return set(range(int(m.group(1)), int(m.group(2)) + 1)) if m else set()


def instructions(asm, name):
    out = []
    for line in kernel_body(asm, name):
        text = line.split(";")[0].strip()
        if text and not text.startswith(".") and not text.endswith(":"):
            out.append(text)
    return out


def operands(text):
    return [o.strip() for o in text.split(None, 1)[1].split(",")] if " " in text or "\t" in text else []


def test_grad_kernels_are_all_there(asm):
    assert len(names(asm, "grad_dma_kernel")) == 3 and len(names(asm, "scaled_dma16_kernel")) == 12


@pytest.mark.parametrize("which", range(3))
def test_mfma_operands_are_two_instructions_old(asm, which):
    code = instructions(asm, names(asm, "grad_dma_kernel")[which])
    mfmas = 0
    for i, text in enumerate(code):
        if not text.startswith("v_mfma_f32_16x16x32_f16"):
            continue
        mfmas += 1
        ops = operands(text)
        assert ops[0].startswith("a[") and ops[0] == ops[3], text
        reads = registers(ops[1]) | registers(ops[2])
        gap, k = 0, i - 1
        while gap < 2 and k >= 0:
            before = code[k]
            if before.startswith("v_") and not before.startswith("v_mfma"):
                assert not registers(operands(before)[0]) & reads, (before, text)
            m = re.match(r"s_nop (\d+)", before)
            gap += int(m.group(1)) + 1 if m else 1
            k -= 1
    rows = int(re.search(r"grad_dma_kernelILi(\d+)E", names(asm, "grad_dma_kernel")[which]).group(1))
    assert mfmas == rows // 2      # one slice's two halves, in the loop


@pytest.mark.parametrize("which", range(3))
def test_nothing_else_in_the_loop_waits_for_vector_memory(asm, which):
    code = instructions(asm, names(asm, "grad_dma_kernel")[which])
    at = [i for i, t in enumerate(code) if t.startswith("v_mfma_f32_16x16x32_f16")]
    loop = code[at[0]:at[-1] + 1]
    waits = [t for t in loop if "vmcnt" in t]
    assert len(waits) == 1, waits
    assert not [t for t in loop if t.startswith(("scratch_", "buffer_", "global_store", "flat_"))]
    m0_belongs_to_dmas(code)


def m0_belongs_to_dmas(code):
    for i, t in enumerate(code):
        if re.search(r"\bm0\b", t):
            assert t.startswith("s_mov_b32 m0,"), t
            assert code[i + 1].startswith("s_nop") and code[i + 2].startswith("global_load_lds_dwordx4"), code[i:i + 3]


@pytest.mark.parametrize("which", range(12))
def test_the_int8_k_loop_is_undisturbed(asm, which):
    code = instructions(asm, names(asm, "scaled_dma16_kernel")[which])
    at = [i for i, t in enumerate(code) if t.startswith("v_mfma_i32_16x16x64_i8")]
    loop = code[at[0]:at[-1] + 1]
    assert len(at) in (256, 128)               # four steps of 64 or 32
    assert len([t for t in loop if "vmcnt" in t]) == 3 and "vmcnt" in " ".join(code[at[-1]:at[-1] + 12])
    assert not [t for t in loop if t.startswith(("scratch_", "buffer_", "global_store", "flat_", "v_accvgpr"))]
    m0_belongs_to_dmas(code)


@pytest.mark.parametrize("which", range(3))
def test_accumulators_stay_in_place(asm, which):
    """Between the first and the last MFMA no accumulator is copied or read."""
    code = instructions(asm, names(asm, "grad_dma_kernel")[which])
    at = [i for i, t in enumerate(code) if t.startswith("v_mfma_f32_16x16x32_f16")]
    assert not [t for t in code[at[0]:at[-1]] if t.startswith("v_accvgpr")]
