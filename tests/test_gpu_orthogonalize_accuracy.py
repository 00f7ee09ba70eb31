"""Orthogonalisation where roundings have most to say: matrices of few directions, which the iteration amplifies what it leaves
in the others of, and equal rows or entries, whose roundings do not average out.  Results in f16, which hide least."""
import pytest
import torch

import layer_ops as L

pytestmark = pytest.mark.gpu


def bound(rows, cols, steps, repeats, out):
    """The error that the header allows (with 2^-23 for what directions that X lacks get, half of the header's), and one rounding to the result's type."""
    base = 3e-3 if steps <= 6 else 6e-3
    few = 4 if repeats or min(rows, cols) < 16 else 1
    return base * few + 2.0**-23 * L.COEFFICIENTS[0]**steps + L.ROUND[out][0]


def matrix(kind, rows, cols, seed):
    g = torch.Generator().manual_seed(1000 * rows + cols + seed)
    new = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if kind.startswith("rank"):
        r = min(int(kind.split()[1]), rows, cols)
        return new(rows, r) @ new(r, cols)
    if kind == "low rank and noise":
        return new(rows, 8) @ new(8, cols) + 1e-3 * new(rows, cols)
    if kind == "one direction above noise":
        return new(rows, cols) + 30 * new(rows, 1) @ new(1, cols)
    if kind == "two equal rows":
        x = torch.zeros(rows, cols)
        x[0] = x[-1] = new(cols)
        return x
    if kind == "equal entries":
        return torch.full((rows, cols), 0.37)
    return new(rows, cols)


# one workgroup a matrix; products on tiles
SHAPES = [(2, 2), (2, 4), (8, 64), (64, 8), (64, 64), (30, 500), (100, 128), (128, 256), (250, 100),
          (2, 600), (33, 600), (600, 33), (64, 520), (130, 520), (300, 700), (700, 300)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("kind", ["rank 1", "rank 2", "rank 4", "low rank and noise", "one direction above noise", "two equal rows", "equal entries"])
def test_few_directions(gpu_handle, rows, cols, kind):
    x = torch.stack([matrix(kind, rows, cols, seed) for seed in range(4)])
    got, want = L.gpu_orthogonalize(gpu_handle, x, "f32", "f16"), L.orthogonalize_plain(x, 5)
    for i in range(4):
        off = L.relative(got[i], want[i])
        assert off <= bound(rows, cols, 5, "equal" in kind, "f16"), (i, off)


@pytest.mark.parametrize("rows,cols", [(2, 4), (8, 64), (64, 64), (128, 256), (100, 50), (33, 600), (300, 200), (512, 512)])
@pytest.mark.parametrize("kind", ["gaussian", "rank 1", "low rank and noise", "two equal rows"])
@pytest.mark.parametrize("steps", [1, 2, 3, 6, 8, 10, 12])
def test_steps(gpu_handle, rows, cols, kind, steps):
    """Results of odd and even numbers of steps, and of more than the usual five or six."""
    x = torch.stack([matrix(kind, rows, cols, 10 + seed) for seed in range(2)])
    got, want = L.gpu_orthogonalize(gpu_handle, x, "f32", "f16", steps), L.orthogonalize_plain(x, steps)
    for i in range(2):
        off = L.relative(got[i], want[i])
        assert off <= bound(rows, cols, steps, "equal" in kind, "f16"), (i, off)


@pytest.mark.parametrize("rows,cols", [(60, 100), (100, 60), (40, 700)])
def test_steps_that_converge(gpu_handle, rows, cols):
    """Coefficients whose error does not grow, and more steps than one launch of a small matrix holds."""
    coefficients = [1.875, -1.25, 0.375]
    x = torch.stack([matrix("gaussian", rows, cols, 20 + seed) for seed in range(2)])
    for steps in (16, 17, 30):
        got, want = L.gpu_orthogonalize(gpu_handle, x, "f32", "f16", steps, coefficients * steps), L.orthogonalize_plain(x, steps, coefficients * steps)
        assert L.relative(got, want) <= 3e-3 + L.ROUND["f16"][0], steps


# steps whose A or B has entries of 64 and more, while no singular value of an iterate reaches 16
GROWING = {"A of up to 225": [15.0, 0.0, 0.0, 1.0, -0.01, 1e-5], "B of up to 130": [-118.0, 130.0, 0.0],
           "A back to 1": [15.0, 0.0, 0.0, 1.0 / 15, 0.0, 0.0, 1.5, -0.5, 0.0]}


@pytest.mark.parametrize("rows,cols", [(2, 4), (64, 64), (128, 256), (100, 20), (2, 600), (600, 2), (33, 600), (300, 200)])
@pytest.mark.parametrize("name", GROWING)
def test_coefficients_that_grow(gpu_handle, rows, cols, name):
    """Of equal entries, so that A and B have entries near their singular value: the tolerance follows that one value s.  X_hi, A' and B' are rounded by up to
    2^-11 of themselves, all entries alike; X_hi is four times in A A X and twice in A X beside the X that B multiplies, A' twice and once, B' once."""
    coefficients = GROWING[name]
    x = torch.full((2, rows, cols), 0.37)
    s, off, u = 1.0, 0.0, 2.0**-11
    for i in range(0, len(coefficients), 3):
        a, b, c = coefficients[i:i + 3]
        grown = abs(a + 3 * b * s**2 + 5 * c * s**4) * off + u * (5 * abs(b) * s**3 + 8 * abs(c) * s**5)
        s, off = a * s + b * s**3 + c * s**5, grown
        assert abs(s) < 16
    steps = len(coefficients) // 3
    want = L.orthogonalize_plain(x, steps, coefficients)
    assert abs(float(want[0, 0, 0]) - s / (rows * cols)**0.5) < 1e-3 * abs(s)
    for out in ("bf16", "f16"):
        got = L.gpu_orthogonalize(gpu_handle, x, "f32", out, steps, coefficients)
        assert L.relative(got, want) <= off / abs(s) + L.ROUND[out][0], (s, off)
