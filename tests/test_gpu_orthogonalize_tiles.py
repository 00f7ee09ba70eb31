"""Orthogonalisation on every tile that its products have, each named, in both orientations, and the rest of its range on more than one workgroup."""
import pytest
import torch

import layer_kernels
import layer_ops as L
from test_gpu_orthogonalize_accuracy import bound

pytestmark = pytest.mark.gpu

# tiles of square, mix and update: (batch, rows, cols); the matrix and its transpose
TILES = {"64_64_64": (2, 150, 301), "64_64_64r2": (1, 1000, 2731), "sliced_64_64": (4, 40, 6047), "sliced_64_64r2": (12, 20, 2704),
         "sliced_64_128": (1, 500, 8000), "sliced_64_192": (4, 130, 8233), "64r2_64r2_128": (16, 449, 451), "128_128_128": (16, 577, 590),
         "128_128_192": (1, 2999, 3001), "128_128_256": (16, 769, 770), "192_192_256": (16, 897, 901), "256_256_128": (16, 1153, 1154)}
TURNED = [(name, turned) for name in TILES for turned in (False, True)]


def shape_of(name, turned):
    batch, rows, cols = TILES[name]
    return (batch, cols, rows) if turned else (batch, rows, cols)


def plain(x, steps, coefficients=None, epsilon=1e-7):
    """The plain form in 64 bits, on the device."""
    out = []
    for y in x:
        y = y.cuda().double()
        y = y / (torch.linalg.norm(y) + epsilon)
        y = y.t().contiguous() if y.shape[0] > y.shape[1] else y
        for i in range(steps):
            a, b, c = coefficients[3 * i:3 * i + 3] if coefficients else L.COEFFICIENTS
            s = y @ y.t()
            y = a * y + (b * s + c * (s @ s)) @ y
        out.append((y.t() if y.shape != x.shape[1:] else y).cpu())
    return torch.stack(out)


def test_plain_form_is_the_other_one():
    x = torch.randn(2, 30, 50, generator=torch.Generator().manual_seed(0))
    for y in (x, x.transpose(1, 2).contiguous()):
        assert (plain(y, 5) - L.orthogonalize_plain(y, 5)).abs().max() < 1e-11


@pytest.mark.parametrize("name,turned", TURNED)
def test_tiles(gpu_handle, name, turned):
    """Odd and even numbers of steps (X changes places with every one), rows with and without gaps on both sides, in place; twice the same."""
    batch, rows, cols = shape_of(name, turned)
    g = torch.Generator().manual_seed(rows + 3 * cols)
    x = torch.randn(batch, rows, cols, generator=g) + torch.randn(batch, rows, 1, generator=g) @ torch.randn(batch, 1, cols, generator=g)
    x = (x * 10.0 ** torch.randint(-4, 3, (batch, 1, 1), generator=g)).bfloat16()
    for steps, out, kw in ((1, "f16", {}), (2, "f16", {"ldx": cols + 3}), (5, "f16", {"ldo": cols + 5}), (5, "bf16", {"in_place": True, "ldx": cols + 8}),
                           (6, "bf16", {"ldx": cols + 8, "ldo": cols + 1})):
        assert layer_kernels.orthogonalize(batch, rows, cols, steps) == "newton_schulz_products_" + name
        want = plain(x, steps)
        got = [L.gpu_orthogonalize(gpu_handle, x, "bf16", out, steps, **kw).clone() for _ in range(2)]
        assert torch.equal(got[0], got[1]), (steps, kw)
        for i in range(batch):
            off = L.relative(got[0][i], want[i])
            assert off <= bound(rows, cols, steps, False, out), (steps, kw, i, off)
            # (no part of a matrix is off: a tile, or the ragged edge of one, would hide in the whole)
            d, whole = got[0][i].double() - want[i], want[i].norm(dim=1, keepdim=True)
            worst = float((d.norm(dim=1, keepdim=True) / whole).max())
            assert worst <= 8 * bound(rows, cols, steps, False, out), (steps, kw, i, worst)


LARGE = [(2, 150, 301), (2, 301, 150), (4, 40, 6047), (3, 6047, 40)]


@pytest.mark.parametrize("batch,rows,cols", LARGE)
def test_coefficients_of_each_step(gpu_handle, batch, rows, cols):
    x = torch.randn(batch, rows, cols, generator=torch.Generator().manual_seed(rows)).bfloat16()
    for steps, coefficients in ((1, [1.5, -0.5, 0.0]), (3, [1.875, -1.25, 0.375] * 3), (4, [3.4445, -4.775, 2.0315, 1.5, -0.5, 0.0] * 2)):
        got = L.gpu_orthogonalize(gpu_handle, x, "bf16", "f16", steps, coefficients)
        assert L.relative(got, plain(x, steps, coefficients)) <= bound(rows, cols, steps, False, "f16"), steps


@pytest.mark.parametrize("batch,rows,cols", LARGE)
def test_extremes_of_large_matrices(gpu_handle, batch, rows, cols):
    """Matrices of zeros, of values whose squares are no f32, of a NaN or an infinity: each keeps to itself."""
    x = torch.randn(batch, rows, cols, generator=torch.Generator().manual_seed(cols))
    x[1] = 0
    for scale, epsilon in ((1e-30, 0.0), (1e30, 1e-7)):
        got, want = L.gpu_orthogonalize(gpu_handle, x * scale, "f32", epsilon=epsilon), plain(x * scale, 5, epsilon=epsilon)
        assert L.relative(got[0], want[0]) <= bound(rows, cols, 5, False, "bf16")
        assert got[1].isnan().all() if epsilon == 0 else (got[1] == 0).all()
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = x.clone()
        y[batch - 1, rows - 1, cols - 1] = bad
        got = L.gpu_orthogonalize(gpu_handle, y, "f32")
        assert got[batch - 1].isnan().all() and not got[:batch - 1].isnan().any()
