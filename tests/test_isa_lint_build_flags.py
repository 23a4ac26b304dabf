"""The ISA lint (tests/test_isa_lint.py) on the instructions of the library that is built: its checks again, with the build's own compiler flags, and
no packed fp32 instruction in any of them."""
import os
import re
import subprocess

import pytest

from open_flamingo_amd.csrc import build
from tests import test_isa_lint as lint

pytestmark = pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc to cross-compile")


@pytest.fixture(scope="module")
def isa(tmp_path_factory):
    made = {}

    def compile_to_asm(src, out=None):
        if src not in made:
            made[src] = str(tmp_path_factory.mktemp("isa") / (src + ".s"))
            subprocess.run(["/opt/rocm/bin/hipcc"] + build.FLAGS + ["-S", "--cuda-device-only", os.path.join(build.HERE, src), "-o", made[src]], check=True, capture_output=True)
        if out is not None:
            os.symlink(made[src], out)
        return made[src]
    return compile_to_asm


@pytest.fixture
def with_build_flags(monkeypatch, isa):
    monkeypatch.setattr(lint, "_compile_to_asm", isa)


@pytest.mark.parametrize("src,min_mfma", lint.ASM_MFMA_SOURCES)
def test_no_valu_write_right_in_front_of_an_asm_mfma(tmp_path, with_build_flags, src, min_mfma):
    lint.test_no_valu_write_right_in_front_of_an_asm_mfma(tmp_path, src, min_mfma)


@pytest.mark.parametrize("src", [s for s, _ in lint.ASM_MFMA_SOURCES if s != "attn_bwd_res.hip"])
def test_accumulators_of_asm_mfmas_are_read_only_after_the_settle_wait(tmp_path, with_build_flags, src):
    lint.test_accumulators_of_asm_mfmas_are_read_only_after_the_settle_wait(tmp_path, src)


@pytest.mark.parametrize("src", ["gemm_w4m.hip", "gemm_w4h.hip", "gemm_w4s.hip", "gemm_mid.hip", "gemm_pp.hip", "attention.hip"])
def test_m0_is_only_ever_the_lds_dma_destination(tmp_path, with_build_flags, src):
    lint.test_m0_is_only_ever_the_lds_dma_destination(tmp_path, src)


def test_nothing_of_the_compilers_lives_in_the_fixed_accumulator_bank(tmp_path, with_build_flags):
    lint.test_nothing_of_the_compilers_lives_in_the_fixed_accumulator_bank(tmp_path)


@pytest.mark.parametrize("src", ["gemm_w4m.hip", "attn_bwd_res.hip", "attention.hip", "xattn_fused.hip", "layernorm.hip", "optim.hip", "linear_ce.hip", "embedding.hip", "optim_multi.hip"])
def test_no_packed_fp32_instruction(isa, src):
    packed = [line for line in open(isa(src)) if re.search(r"\bv_pk_(add|mul|fma)_f32\b", line)]
    assert not packed, (len(packed), packed[:3])
