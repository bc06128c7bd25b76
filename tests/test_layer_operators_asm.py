"""Compiled code of the loss' and adapters' kernels whose k loops are inline assembly (test_scaled_asm.py says what
such a loop may hold), and of the low-rank products written as inline assembly themselves."""
import os
import re
import subprocess

import pytest

from test_scaled_asm import m0_belongs_to_dmas, operands, registers
from veritac_amd import _lib

BIN = "/opt/rocm/llvm/bin/"


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    """The built library's kernels as {name: instructions} (disassembled: a second compilation takes minutes)."""
    folder = tmp_path_factory.mktemp("code")
    fat, code = str(folder / "fat"), str(folder / "code.o")
    subprocess.run([BIN + "llvm-objcopy", "--dump-section", ".hip_fatbin=" + fat, _lib.library_path(), os.devnull], check=True)
    listed = subprocess.run([BIN + "clang-offload-bundler", "--list", "--type=o", "--input=" + fat], check=True, capture_output=True, text=True)
    target = next(t for t in listed.stdout.split() if "gfx950" in t)
    subprocess.run([BIN + "clang-offload-bundler", "--unbundle", "--type=o", "--input=" + fat, "--targets=" + target, "--output=" + code], check=True)
    text = subprocess.run([BIN + "llvm-objdump", "-d", "--no-show-raw-insn", "--no-leading-addr", code], check=True, capture_output=True,
                          text=True).stdout
    kernels, now = {}, None
    for line in text.splitlines():
        m = re.match(r"(?:[0-9a-f]+ )?<(\S+)>:", line)
        if m:
            now = kernels.setdefault(m.group(1), [])
        elif now is not None and line.strip():
            now.append(re.sub(r"\s+", " ", line.split("//")[0]).strip())
    return kernels


def names(asm, kernel):
    return sorted(n for n in asm if re.match(r"_Z\S*%s" % kernel, n) and not n.endswith(".kd"))


def instructions(asm, name):
    return asm[name]

TILES = 3 + 2 * 3      # adapted outputs of three types on one tile; the loss and its terms, in one and two halves, on two


def test_all_are_there(asm):
    assert len(names(asm, "out_dma16_kernel")) == TILES and len(names(asm, "adapted_dx_kernel")) == 9


@pytest.mark.parametrize("which", range(TILES))
def test_the_int8_k_loop_is_undisturbed(asm, which):
    code = instructions(asm, names(asm, "out_dma16_kernel")[which])
    at = [i for i, t in enumerate(code) if t.startswith("v_mfma_i32_16x16x64_i8")]
    loop = code[at[0]:at[-1] + 1]
    assert len(at) in (256, 128)
    assert len([t for t in loop if "vmcnt" in t]) == 3 and "vmcnt" in " ".join(code[at[-1]:at[-1] + 12])
    assert not [t for t in loop if t.startswith(("scratch_", "buffer_", "global_store", "flat_", "v_accvgpr"))]
    m0_belongs_to_dmas(code)


@pytest.mark.parametrize("which", range(9))
def test_the_gradient_s_loop_is_undisturbed(asm, which):
    name = names(asm, "adapted_dx_kernel")[which]
    code = instructions(asm, name)
    at = [i for i, t in enumerate(code) if t.startswith("v_mfma_f32_16x16x32_f16") and operands(t)[0].startswith("a[")]
    rows = int(re.search(r"adapted_dx_kernelILi\dELi(\d+)E", name).group(1))
    assert len(at) == rows // 2
    loop = code[at[0]:at[-1] + 1]
    assert len([t for t in loop if "vmcnt" in t]) == 1
    assert not [t for t in loop if t.startswith(("scratch_", "buffer_", "global_store", "flat_", "v_accvgpr"))]
    m0_belongs_to_dmas(code)
    for i in at:
        ops = operands(code[i])
        assert ops[0] == ops[3]
        reads, gap, k = registers(ops[1]) | registers(ops[2]), 0, i - 1
        while gap < 2 and k >= 0:
            if code[k].startswith("v_") and not code[k].startswith("v_mfma"):
                assert not registers(operands(code[k])[0]) & reads, (code[k], code[i])
            m = re.match(r"s_nop (\d+)", code[k])
            gap += int(m.group(1)) + 1 if m else 1
            k -= 1


@pytest.mark.parametrize("kernel,count", [("out_dma16_kernelINS_11AdaptedTile", 3), ("adapted_dx_kernel", 9),
                                          ("gemm_mfma_kernelI\\S*AdaptedTile", 9)])
def test_low_rank_products_wait_for_themselves(asm, kernel, count):
    """Products into VGPRs: two wait states before a run of them, 24 after it, and four apart on the same sums."""
    found = names(asm, kernel)
    assert len(found) == count
    for name in found:
        code = instructions(asm, name)
        low = [i for i, t in enumerate(code) if re.match("v_mfma_f32_16x16x(4_f32|32_bf16|32_f16) v", t)]
        assert low
        for i in low:
            ops = operands(code[i])
            assert ops[0] == ops[3] and ops[0].startswith("v[")
            if i - 1 not in low:
                assert code[i - 1] == "s_nop 1", code[i - 1:i + 1]
            if i + 1 not in low:
                assert code[i + 1:i + 3] == ["s_nop 15", "s_nop 7"], code[i:i + 3]
            for k in range(i - 3, i):
                if k in low:
                    assert operands(code[k])[0] != ops[0], code[k:i + 1]


def test_u_and_the_adapters_gradients_do_not_spill(asm):
    """Workgroups of 16 waves have 128 registers a lane: their loads in flight are chosen to fit."""
    kernels = names(asm, "shrink_tiles_kernel") + names(asm, "shrink_rows_kernel") + names(asm, "outer_kernel")
    assert len(kernels) >= 20
    assert not [n for n in kernels if any(t.startswith("scratch_") for t in instructions(asm, n))]
