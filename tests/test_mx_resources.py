"""What the compiler reports for the kernels over MXFP4 pages and those on pages
and logits: registers that are not spilled, workgroups that fit a CU."""
import pytest

from test_kernel_resources import _kernels


@pytest.fixture(scope="module")
def kernels(yl):
    return _kernels(yl.LIB_PATH)


def test_single_row_and_row_kernels_keep_their_registers(kernels):
    mine = {n: k for n, k in kernels.items() if "k_paged_attn_few" in n or ("k_paged_attn_rows" in n and "Mx4" in n)}
    assert len(mine) == 9
    spilled = {n: k[".vgpr_spill_count"] for n, k in mine.items() if k[".vgpr_spill_count"]}
    assert not spilled, spilled


def test_tile_kernels_spill_nothing_that_their_loop_needs(kernels):
    # head size 64: four wavefronts per SIMD leave 128 registers; five hold what is wanted before and behind the loop, and
    # once in 16 of its steps
    mine = {n: k[".vgpr_spill_count"] for n, k in kernels.items() if "k_paged_attn_tile" in n and "Mx4" in n}
    assert len(mine) == 3 and all(v <= 5 for v in mine.values()), mine


def test_kernels_on_pages_and_logits(kernels):
    mine = {n: k for n, k in kernels.items() if "k_pages_" in n or "k_logit_rules" in n or "k_paged_gather" in n}
    assert len(mine) >= 20
    assert all(not k[".vgpr_spill_count"] and not k[".private_segment_fixed_size"] for k in mine.values())
    # four workgroups of 512 threads, and of the rules' LDS, on a CU
    assert all(k[".group_segment_fixed_size"] <= 40960 for n, k in mine.items() if "k_logit_rules" in n)
