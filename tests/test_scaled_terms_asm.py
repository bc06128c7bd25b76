"""Compiled code of terms_low_dma16_kernel (gradient terms with low halves on the persistent tiles): the
k loop that scaled_dma16_kernel's checks describe, in front of an epilogue of its own."""
import pytest

from test_dma_asm import asm  # noqa: F401
from test_scaled_asm import instructions, m0_belongs_to_dmas, names


def test_both_tile_widths_are_there(asm):
    assert len(names(asm, "terms_low_dma16_kernel")) == 2


@pytest.mark.parametrize("which", range(2))
def test_the_int8_k_loop_is_undisturbed(asm, which):
    code = instructions(asm, names(asm, "terms_low_dma16_kernel")[which])
    at = [i for i, t in enumerate(code) if t.startswith("v_mfma_i32_16x16x64_i8")]
    loop = code[at[0]:at[-1] + 1]
    assert len(at) in (256, 128)
    assert len([t for t in loop if "vmcnt" in t]) == 3 and "vmcnt" in " ".join(code[at[-1]:at[-1] + 12])
    assert not [t for t in loop if t.startswith(("scratch_", "buffer_", "global_store", "flat_", "v_accvgpr"))]
    m0_belongs_to_dmas(code)
