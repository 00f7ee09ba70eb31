"""Layer operators at sizes that the other tests do not reach."""
import pytest
import torch

import layer_kernels
import layer_ops as L
from hiptensor_amd import api

pytestmark = pytest.mark.gpu


def test_one_token_and_more_columns_than_a_grid_of_few_tokens_holds(gpu_handle):
    """N of 2^27 and more (B of 2 GiB), in tiles."""
    n, k = (1 << 27) + 21, 16
    assert "few" not in layer_kernels.product(1, n, k, 128, "bf16")
    g = torch.Generator(device="cuda").manual_seed(3)
    b = torch.randint(0, 256, (n, k), dtype=torch.uint8, device="cuda", generator=g) & 0xB7  # (no NaN among these)
    a = torch.randint(0, 256, (1, k), dtype=torch.uint8, device="cuda", generator=g) & 0xB7
    sa = torch.full((1, 1), 0.25, device="cuda")
    sb = torch.rand(1, L.blocks(n), device="cuda", generator=g) + 0.5
    d = torch.empty(1, n, dtype=torch.bfloat16, device="cuda")
    api.check(api.hiptensorBlockScaledProduct(gpu_handle, 1, n, k, 1.0, a.data_ptr(), k, sa.data_ptr(), 1, b.data_ptr(), k, sb.data_ptr(), sb.shape[1], 128, 0.0,
                                              None, d.data_ptr(), api.HIP_R_16BF, n, None, 0, L.stream()))
    va = a.view(torch.float8_e4m3fn).float() * 0.25
    for at in range(0, n, 1 << 24):
        rows = slice(at, min(n, at + (1 << 24)))
        scale = sb[0, torch.arange(rows.start, rows.stop, device="cuda") // 128]
        terms = b[rows].view(torch.float8_e4m3fn).float() * va * scale[:, None]
        want, most = terms.sum(1), terms.abs().sum(1)
        assert ((d[0, rows].float() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-10 * most).all(), at


def test_small_orthogonalisation_without_a_workspace(gpu_handle):
    x = torch.randn(3, 60, 200, generator=torch.Generator().manual_seed(4))
    want = L.gpu_orthogonalize(gpu_handle, x, "f32")
    dx, o = x.cuda(), torch.empty(3, 60, 200, dtype=torch.bfloat16, device="cuda")
    api.check(api.hiptensorOrthogonalize(gpu_handle, 3, 60, 200, dx.data_ptr(), api.HIP_R_32F, 200, 12000, 5, None, 1e-7, o.data_ptr(), api.HIP_R_16BF, 200,
                                         12000, None, 0, L.stream()))
    assert torch.equal(o.cpu(), want)
