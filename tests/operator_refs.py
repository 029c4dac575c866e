"""64-bit references of the operators beyond plain attention, and the tolerances that go with them.

Attention.  The kernels sum the softmax in fp32, round the unnormalised weights P to bf16 for the second
product (the row sum takes them unrounded) and the result to bf16.  bf16 rounds by at most 2^-8 of the
value, so with A = sum_j p_j |v_j| (p normalised)
    |out - ref| <= 2^-8 A + 2^-8 |ref| + d A .
d covers the scores' own errors, which shift exponents: the fp32 products (a few 1e-5 at |s| of some tens),
the tanh (cap * 2.8e-6 <= 1.5e-4 natural-log units at cap 50), exp2 (2^-22), each entering numerator and
denominator: d = 1e-3 is above all of them together.  The LSE has the same shift and no rounding to bf16:
1e-3 absolute, the bar of the plain kernels.

Projection.  q - z is exact in bf16, products are exact in fp32, the sum over K inputs is off by at most a
few K 2^-24 of B = sum |x| |w| (fp32 with a handful of roundings per 16 inputs): 2e-5 B at the sizes here.
Above 16 rows the weights themselves are rounded to bf16 first: 2^-8 B more.
"""
import numpy as np
import torch

F64 = torch.float64
HALF_BF16 = 2.0 ** -8


def attention_ref(q, k, v, lo, hi, pos, scale, cap=0.0, slopes=None, shared=0):
    """q [rows, H, D]; k, v [Hkv, L, D]; lo, hi, pos [rows] (key indices; `shared` keys come first and are seen by
    all rows).  Returns out, A [rows, H, D] and lse [rows, H], fp64."""
    rows, H, D = q.shape
    dev = q.device
    g = H // k.shape[0]
    kk, vv = k.to(F64).repeat_interleave(g, 0), v.to(F64).repeat_interleave(g, 0)
    s = torch.einsum("rhd,hld->hrl", q.to(F64), torch.nan_to_num(kk, 0.0, 0.0, 0.0)) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    j = torch.arange(k.shape[1], device=dev)
    lo, hi, pos = (torch.as_tensor(np.asarray(x), device=dev) for x in (lo, hi, pos))
    if slopes is not None:
        s = s - slopes.to(F64).view(H, 1, 1) * (pos[:, None] - j).abs()
    seen = ((j >= lo[:, None]) & (j < hi[:, None])) | (j < shared)
    s = s.masked_fill(~seen, float("-inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
    used = seen.any(0)
    vv = torch.where(used[None, :, None], vv, 0.0)
    # a masked key adds nothing whatever its V row holds: products over finite values, visible ones put back
    if bool(torch.isfinite(vv).all()):
        out = torch.einsum("hrl,hld->rhd", p, vv)
        A = torch.einsum("hrl,hld->rhd", p, vv.abs())
    else:
        out = torch.zeros(rows, H, D, dtype=F64, device=dev)
        A = torch.zeros_like(out)
        for r in range(rows):
            idx = seen[r].nonzero().flatten()
            out[r] = torch.einsum("hl,hld->hd", p[:, r, idx], vv[:, idx])
            A[r] = torch.einsum("hl,hld->hd", p[:, r, idx], vv[:, idx].abs())
    return out, A, lse.T


def assert_attention(out, ref, A, lse=None, lse_ref=None):
    out = out.to(F64)
    assert bool(torch.isfinite(out).all()), "non-finite output"
    tol = (HALF_BF16 + 1e-3) * A + HALF_BF16 * ref.abs() + 1e-6
    excess = ((out - ref).abs() / tol).max().item()
    assert excess <= 1.0, f"error is {excess:.3f} of the tolerance"
    if lse is not None:
        empty = torch.isinf(lse_ref)
        assert bool((torch.isneginf(lse) == empty).all())
        assert (lse.to(F64) - lse_ref)[~empty].abs().max().item() <= 1e-3 if bool((~empty).any()) else True


def w4_weights(q, scales, zeros, group):
    z = zeros.to(F64).repeat_interleave(group, 1) if zeros is not None else 8.0
    return (q.to(F64) - z) * scales.to(F64).repeat_interleave(group, 1)


def assert_w4(out, a, w, residual, rounded_weights):
    a64 = a.to(F64)
    ref = a64 @ w.T
    B = a64.abs() @ w.abs().T
    if residual is not None:
        ref = ref + residual.to(F64)
    tol = HALF_BF16 * ref.abs() + 2e-5 * B + (HALF_BF16 * B if rounded_weights else 0.0) + 1e-30
    excess = ((out.to(F64) - ref).abs() / tol).max().item()
    assert excess <= 1.0, f"error is {excess:.3f} of the tolerance"
