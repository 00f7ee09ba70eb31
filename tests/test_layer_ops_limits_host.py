"""Limits and choices of the layer operators that need no device: what is accepted, which kernel a call is for, what the compiler made
of the small orthogonalisation's kernels."""
import re

from test_layer_ops_codegen import kernels


def test_orthogonalisation_in_one_workgroup_does_not_spill(tmp_path):
    found = kernels("newton_schulz", tmp_path, "ns_small_kernel")
    assert len(found) == 6, sorted(found)
    for symbol, body in found.items():
        text = "\n".join(body)
        assert "scratch_" not in text and not re.search(r"vgpr_spill_count:\s+[1-9]", text), symbol
