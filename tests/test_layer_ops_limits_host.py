"""Limits and choices of the layer operators that need no device: what is accepted, which kernel a call is for, what the compiler made
of the small orthogonalisation's kernels."""
import re

import pytest

import layer_kernels
from hiptensor_amd import api
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


def test_matrices_of_one_workgroup_need_no_workspace(host_handle):
    """The size asked for is enough for any number of steps; a call needs what it touches, which is nothing up to 64 x 512 or 128 x 256 and 16 steps."""
    def call(rows, cols, steps, workspace, size, batch=3):
        return api.hiptensorOrthogonalize(host_handle, batch, rows, cols, 1 << 20, api.HIP_R_32F, cols, rows * cols, steps, None, 1e-7, 1 << 20, api.HIP_R_16F,
                                          cols, rows * cols, workspace, size, None)

    ok, small = api.HIPTENSOR_STATUS_ARCH_MISMATCH, api.HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE
    for rows, cols in ((1, 1), (64, 512), (512, 64), (128, 256), (200, 100)):
        need = api.check(api.hiptensorOrthogonalizeGetWorkspaceSize(host_handle, 3, rows, cols, api.HIP_R_32F, api.HIP_R_16F))
        assert call(rows, cols, 5, None, 0) == call(rows, cols, 16, None, 0) == ok
        assert need > 0 and call(rows, cols, 17, None, 0) == call(rows, cols, 17, 1 << 20, need - 1) == small and call(rows, cols, 17, 1 << 20, need) == ok
    for rows, cols in ((65, 257), (64, 513), (129, 129)):
        assert call(rows, cols, 5, None, 0) == small


def test_largest_sizes_that_the_header_names(host_handle):
    """Accepted at the limit (as far as a handle without a device goes), refused one beyond it."""
    ok, invalid, unsupported = api.HIPTENSOR_STATUS_ARCH_MISMATCH, api.HIPTENSOR_STATUS_INVALID_VALUE, api.HIPTENSOR_STATUS_NOT_SUPPORTED
    at, most, tiles = 1 << 20, (1 << 31) - 256, (1 << 23) - 1

    def quantize(rows, cols):
        return api.hiptensorBlockQuantize(host_handle, rows, cols, at, api.HIP_R_16BF, cols, 1, at, cols, at, rows, None, 0, None, 0, None)

    def product(m, n, k):
        return api.hiptensorBlockScaledProduct(host_handle, m, n, k, 1.0, at, k, at, m, at, k, at, n, 1, 0.0, None, at, api.HIP_R_32F, n, None, 0, None)

    def orthogonalize(batch, rows, cols):
        return api.hiptensorOrthogonalize(host_handle, batch, rows, cols, at, api.HIP_R_32F, cols, rows * cols, 5, None, 0.0, at, api.HIP_R_16F, cols,
                                          rows * cols, at << 20, 1 << 60, None)

    assert quantize(1, tiles * 128) == ok and quantize(1, tiles * 128 + 129) == unsupported and quantize(most + 1, 1) == invalid
    assert product(1, tiles * 64, 8) == ok and product(1, tiles * 64 + 65, 8) == unsupported and product(8, 8, most) == ok and product(8, 8, most + 1) == invalid
    assert orthogonalize(65535, 100, 200) == ok and orthogonalize(65536, 100, 200) == invalid
    assert orthogonalize(1, 1 << 16, 1 << 20) == orthogonalize(1, 1 << 20, 1 << 16) == ok
    assert orthogonalize(1, (1 << 16) + 1, 1 << 20) == orthogonalize(1, 1, (1 << 20) + 1) == invalid
