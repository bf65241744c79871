"""The build's check of register counts, on ptxas reports."""

import pytest

from jitcast_b200 import build


def report(*kernels):
    return "\n".join(f"ptxas info    : Compiling entry function '{name}' for 'sm_100a'\n"
                     f"ptxas info    : Function properties for {name}\n"
                     f"    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads\n"
                     f"ptxas info    : Used {n} registers, used 1 barriers" for name, n in kernels)


def tiles(bits, dim, form, regs, t="6__half"):
    return f"_ZN2jc12_GLOBAL__N_122kv_attention_tc_kernelI{t}Li{bits}ELi{dim}ELi{form}EEEv14CUtensorMap_st", regs


GOOD = [tiles(16, 64, 0, 96), tiles(16, 64, 1, 168), tiles(16, 128, 1, 168, "13__nv_bfloat16"), tiles(4, 64, 1, 128),
        tiles(4, 128, 1, 128)]


def test_counts_that_the_kernels_share_out():
    build.check_registers("kv_attention_tc.cu", report(*GOOD))
    build.check_registers("gemm.cu", "")  # a file that asks for none


@pytest.mark.parametrize("i", [1, 2, 3, 4])
def test_another_count_fails_the_build(i):
    name, n = GOOD[i]
    with pytest.raises(RuntimeError, match="registers"):
        build.check_registers("kv_attention_tc.cu", report(*GOOD[:i], (name, n - 8), *GOOD[i + 1:]))


def test_a_report_without_the_kernels_fails_the_build():
    with pytest.raises(RuntimeError):
        build.check_registers("kv_attention_tc.cu", report(GOOD[0]))
