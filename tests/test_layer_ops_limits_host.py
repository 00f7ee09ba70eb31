"""Limits and choices of the layer operators that need no device: what is accepted, which kernel a call is for, what the compiler made
of the small orthogonalisation's kernels."""
import re

import pytest

import layer_kernels
from test_layer_ops_codegen import kernels


def test_orthogonalisation_in_one_workgroup_does_not_spill(tmp_path):
    found = kernels("newton_schulz", tmp_path, "ns_small_kernel")
    assert len(found) == 6, sorted(found)
    for symbol, body in found.items():
        text = "\n".join(body)
        assert "scratch_" not in text and not re.search(r"vgpr_spill_count:\s+[1-9]", text), symbol


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_few_tokens_run_through_registers_only_where_the_grid_holds_them(dtype):
    """A workgroup of 512 threads takes 16 rows of B, and a launch has fewer than 2^31 threads a dimension: wider products take tiles."""
    for m in (1, 2, 40):
        for n in ((1 << 26) - 16, (1 << 26) + 5, 1 << 27, 1 << 28, 1 << 29):
            name = layer_kernels.product(m, n, 16, 128, dtype)
            assert not ("few" in name and (n + 15) // 16 * 512 >= 1 << 31), (m, n, name)
    assert "few" in layer_kernels.product(1, (1 << 26) - 16, 16, 128, dtype)
