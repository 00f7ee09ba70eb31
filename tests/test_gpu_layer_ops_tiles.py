"""Block-scaled products on every tile the library has, each named, so that a rule that is tuned anew cannot drop one from the tests."""
import math

import pytest
import torch

import layer_kernels
import layer_ops as L
from hiptensor_amd import api

pytestmark = pytest.mark.gpu

# name: (M, N, where K begins).  Neither M nor N is a multiple of anything; the K of a case is that of whole blocks and a tail.
TILES = {"block_product_few": (19, 1003, 640), "block_product_64x64": (131, 133, 640), "block_product_64x128": (130, 5491, 640),
         "block_product_128x128": (1288, 5381, 640), "block_product_256x128": (5485, 645, 640), "block_product_256x256": (1282, 5897, 640),
         "block_product_few_f16": (19, 1003, 640), "block_product_64x64_f16": (131, 133, 640), "block_product_128x128_f16": (5441, 515, 640),
         "block_product_256x128_f16": (5153, 789, 1024)}


def types(name):
    return ["f32"] if name.endswith("f16") else ["bf16", "f16"]


def device_values(codes, scales, k, block_rows):
    rows = codes.shape[0]
    s = scales.cuda().double().t().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :k]
    return codes.cuda().view(torch.float8_e4m3fn)[:, :k].double() * s


CASES = [(name, dtype, block_rows) for name in TILES for dtype in types(name) for block_rows in (1, 128)]


@pytest.mark.parametrize("name,dtype,block_rows", CASES)
def test_tile(gpu_handle, name, dtype, block_rows):
    """One block, and more blocks than a ring of stages holds, with tails; onto a C beside D and onto D itself; twice the same.

    Each element within the bound of its sum; and in 2-norm, where losses of single terms show that the bound of a sum of K terms would let pass: one
    rounding to the type (at most 1 / sqrt(3) of its largest) and 5e-5 for sums of the 8-bit instructions, or 1e-6 for sums in f32."""
    m, n, start = TILES[name]
    for k in (40, start + 23, start + 128) if start < 1000 else (start + 23, start + 128):
        if k != 40:
            assert layer_kernels.product(m, n, k, block_rows, dtype) == name
        g = torch.Generator().manual_seed(m + n + k + block_rows)
        a, sa = L.random_codes(m, k, 1, g)
        b, sb = L.random_codes(n, k, block_rows, g)
        c = (torch.randn(m, n, generator=g) * 50).to(L.TORCH[dtype])
        va, vb = device_values(a, sa, k, 1), device_values(b, sb, k, block_rows)
        product, terms = (va @ vb.t()).cpu(), (va.abs() @ vb.abs().t()).cpu()
        norm = L.ROUND[dtype][0] / math.sqrt(3) + (1e-6 if dtype == "f32" else 5e-5)
        for alpha, beta, kw in ((1.0, 0.0, {}), (-1.5, 0.75, {"ldd": n + 3}), (-1.5, 0.75, {"alias": True})):
            want, most = alpha * product + beta * c.double(), abs(alpha) * terms + abs(beta) * c.double().abs()
            got = [L.gpu_product(gpu_handle, a, sa, b, sb, k, block_rows, dtype, alpha, beta, c if beta else None, **kw).clone() for _ in range(2)]
            assert torch.equal(got[0], got[1]), (k, kw)
            off = got[0].double() - want
            assert (off.abs() <= L.product_bound(want, most, k, dtype)).all(), (k, kw)
            assert float(off.norm() / want.norm()) <= norm, (k, kw, float(off.norm() / want.norm()))


@pytest.mark.parametrize("name,dtype,block_rows", CASES)
@pytest.mark.parametrize("tail", [1, 15, 16, 17, 127])
def test_every_term_counts_once(gpu_handle, name, dtype, block_rows, tail):
    """Codes of -1, 0 and 1 with scales of 1 and 2: all sums are whole numbers that every type holds, so the result is that, bit for bit."""
    m, n, start = TILES[name]
    k = start + tail
    assert layer_kernels.product(m, n, k, block_rows, dtype) == name
    g = torch.Generator(device="cuda").manual_seed(tail + block_rows)

    def codes(rows, per):
        ld = -(-k // 16) * 16
        q = torch.full((rows, ld), 0x7F, dtype=torch.uint8, device="cuda")
        u = torch.rand(rows, k, generator=g, device="cuda")
        q[:, :k] = torch.where(u < 0.12, 0x38, torch.where(u < 0.24, 0xB8, 0)).to(torch.uint8)
        # (the last terms of a row are all there)
        q[:, k - 1] = 0x38
        s = 1.0 + (torch.rand(L.blocks(k), L.blocks(rows, per), generator=g, device="cuda") < 0.5).float()
        return q.cpu(), s.cpu()

    a, sa = codes(m, 1)
    b, sb = codes(n, block_rows)
    want = (device_values(a, sa, k, 1) @ device_values(b, sb, k, block_rows).t()).cpu()
    assert want.abs().max() <= 256 and torch.equal(want, want.round())
    got = L.gpu_product(gpu_handle, a, sa, b, sb, k, block_rows, dtype)
    assert torch.equal(got.double(), want)


# (workspace that the library asks for: partial sums of slices of K)
SLICED = [("block_product_64x128", 23, 4096, 8192 + 40, "f16", 128), ("block_product_256x128", 1000, 1030, 16384 + 7, "bf16", 1),
          ("block_product_64x64", 300, 300, 4100, "bf16", 128),
          ("block_product_64x64_f16", 1000, 999, 8192 + 130, "f32", 1)]


@pytest.mark.parametrize("name,m,n,k,dtype,block_rows", SLICED)
def test_slices(gpu_handle, name, m, n, k, dtype, block_rows):
    assert layer_kernels.product(m, n, k, block_rows, dtype) == name
    assert api.check(api.hiptensorBlockScaledProductGetWorkspaceSize(gpu_handle, m, n, k, block_rows, L.TYPE[dtype])) > 0
    g = torch.Generator().manual_seed(m + n + k)
    a, sa = L.random_codes(m, k, 1, g)
    b, sb = L.random_codes(n, k, block_rows, g)
    va, vb = device_values(a, sa, k, 1), device_values(b, sb, k, block_rows)
    # (scales 2^-8 .. 2^-3 on both sides and thousands of terms: held to what f16 has)
    want, terms = (va @ vb.t()).cpu(), (va.abs() @ vb.abs().t()).cpu()
    scale = 0.125
    got = [L.gpu_product(gpu_handle, a, sa, b, sb, k, block_rows, dtype, scale).clone() for _ in range(2)]
    assert torch.equal(got[0], got[1])
    off = got[0].double() - scale * want
    assert (off.abs() <= L.product_bound(scale * want, scale * terms, k, dtype)).all()
    assert float(off.norm() / (scale * want).norm()) <= L.ROUND[dtype][0] / math.sqrt(3) + (1e-6 if dtype == "f32" else 5e-5)
