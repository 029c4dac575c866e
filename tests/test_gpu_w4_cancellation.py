"""4-bit projections where the terms of a sum cancel or vanish: groups whose numbers equal their zero point, a few numbers
that differ from it, zero points up to 127, rows of one sign with a large common offset.  Every kernel multiplies q - z (or
(q - z) * scale rounded to bf16), so a weight of zero adds exactly nothing and the error of a sum is that of its own terms:

  * a product of two bf16 numbers is exact in fp32;
  * sums are formed 16 inputs at a time (one product step, a handful of roundings of 2^-24 or truncations of 2^-23 of at
    most B = sum |x| |w|), each group's is scaled and added: another two.  Steps and groups of zeros round nothing.  The
    kernels may take the inputs of a 32-block in any order, so a 32-block with a weight counts as two steps.  With s steps
    and groups that hold a weight the sum is off by at most 4 s 2^-23 B;
  * a residual is added with one more rounding and the result is rounded to bf16 once: (2^-8 + 2^-22) |value|;
  * above 32 rows the weights are ((q - z) * scale) rounded to bf16, and that is what the reference multiplies by."""
import pytest
import torch

DEV = "cuda:0"
# (rows, kernel): the warp-level and the tensor-memory form of few rows, the latter with 32, and many rows
FORMS = [(1, 0), (8, 0), (16, 0), (3, 1), (16, 1), (32, -1), (40, -1), (300, -1)]


def weights(q, scales, z, group, rows):
    w = (q.double() - z.double().repeat_interleave(group, 1)) * scales.double().repeat_interleave(group, 1)
    return w.to(torch.bfloat16).double() if rows > 32 else w


def run(q, scales, z, a, residual, group, kernel):
    from ellm_b200 import MatMulAddW4, pack_int4
    rows, (n, k) = a.shape[0], q.shape
    q, scales, z, a = (t.to(DEV) for t in (q, scales, z, a))
    r = residual.to(DEV) if residual is not None else None
    out = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device=DEV)
    op = MatMulAddW4.new(a, pack_int4(q), scales, r, out, rows, n, k, group, zeros=z)
    op.set_pairing(kernel)
    op.run(0, 1, rows)
    torch.cuda.synchronize()
    op.close()
    return out, a, weights(q, scales, z, group, rows), r


def assert_sum(out, a, w, residual, group):
    a64, n, k = a.double(), *w.shape
    live = lambda size: (w.view(n, k // size, size) != 0).any(2).sum(1).double()   # noqa: E731
    s = 2 * live(32) + live(group)
    ref = a64 @ w.T + (0.0 if residual is None else residual.double())
    tol = 4 * 2.0 ** -23 * s * (a64.abs() @ w.abs().T) + (2.0 ** -8 + 2.0 ** -22) * ref.abs()
    assert bool(((out.double() - ref).abs() <= tol).all()), f"error is {((out.double() - ref).abs() / (tol + 1e-30)).max().item():.3f} of the tolerance"


def rows_of(kind, rows, k, g):
    a = torch.randn(rows, k, generator=g)
    if kind == "one sign":
        a = a.abs() + 1.0
    elif kind == "offset":
        a = a + 60.0
    return a.to(torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,kernel", FORMS, ids=str)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", ["normal", "offset"])
def test_columns_whose_numbers_are_their_zero_points_add_nothing(rows, kernel, group, kind):
    g = torch.Generator().manual_seed(1)
    n, k = 264, 1024
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8)
    q = z.repeat_interleave(group, 1)
    scales = (torch.rand(n, k // group, generator=g) + 0.5).to(torch.bfloat16)
    res = torch.randn(rows, n, generator=g).to(torch.bfloat16)
    out, _, _, r = run(q, scales, z, rows_of(kind, rows, k, g), res, group, kernel)
    assert torch.equal(out, r)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,kernel", FORMS, ids=str)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("top", [15, 127])
@pytest.mark.parametrize("kind", ["normal", "one sign", "offset"])
def test_few_numbers_differ_from_their_zero_point(rows, kernel, group, top, kind):
    """Most of a column is at its zero point; where a zero point is past 15, no number can be."""
    g = torch.Generator().manual_seed(2)
    n, k = 136, 1024
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8)
    q = z.repeat_interleave(group, 1).clone()
    at = torch.randint(0, k, (n, 3), generator=g)
    q.scatter_(1, at, torch.randint(0, 16, (n, 3), generator=g, dtype=torch.uint8))
    if top > 15:
        z[::5, 1] = torch.randint(100, 128, (len(z[::5]),), generator=g, dtype=torch.uint8)
    scales = (torch.rand(n, k // group, generator=g) + 0.5).to(torch.bfloat16)
    out, a, w, _ = run(q, scales, z, rows_of(kind, rows, k, g), None, group, kernel)
    assert_sum(out, a, w, None, group)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,kernel", FORMS, ids=str)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", ["normal", "one sign"])
def test_any_numbers_and_zero_points(rows, kernel, group, kind):
    """All numbers and zero points 0..127 at random, a tail of columns, every group's own scale."""
    g = torch.Generator().manual_seed(3)
    n, k = 200, 768
    q = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    z = torch.randint(0, 128, (n, k // group), generator=g, dtype=torch.uint8)
    scales = ((torch.rand(n, k // group, generator=g) + 0.5) * 0.1).to(torch.bfloat16)
    res = torch.randn(rows, n, generator=g).to(torch.bfloat16)
    out, a, w, r = run(q, scales, z, rows_of(kind, rows, k, g), res, group, kernel)
    assert_sum(out, a, w, r, group)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 300])
def test_extreme_weights_of_many_rows_are_exact(rows):
    """One-hot rows, zero points 0 to 127: (q - z) * 3 is exact in bf16 up to 256 and is what comes out."""
    n, k = 40, 128
    q = (torch.arange(n)[:, None] + torch.arange(k)[None]).remainder(16).to(torch.uint8)
    scales = torch.full((n, 4), 3.0, dtype=torch.bfloat16)
    z = torch.tensor([0, 15, 8, 127], dtype=torch.uint8).repeat(n, 1)
    a = torch.zeros(rows, k, dtype=torch.bfloat16)
    a[torch.arange(rows), torch.arange(rows) % k] = 1.0
    out, a, w, _ = run(q, scales, z, a, None, 32, -1)
    assert torch.equal(out, (a.double() @ w.T).to(torch.bfloat16))
