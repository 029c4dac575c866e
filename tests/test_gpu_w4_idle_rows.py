"""A 4-bit projection made for many sequences that runs a few: rows behind the last live one take no part in the choice of
the kernel, nor of how the weights are rounded."""
import pytest
import torch

from operator_refs import HALF_BF16, w4_weights
from test_gpu_w4 import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_batch", [40, 64, 300])
@pytest.mark.parametrize("live", [1, 9, 16, 17, 32])
@pytest.mark.parametrize("intervals", [1, 3])
def test_few_live_rows_give_the_bits_of_a_handle_made_for_them(max_batch, live, intervals):
    from ellm_b200 import MatMulAddW4, pack_int4
    n, k, group = 264, 1024, 64
    q, scales, z, a, r = make(121, intervals * max_batch, n, k, group, True, True)
    a = (a.view(intervals, max_batch, k) * 4.0 + 3.0).to(torch.bfloat16)
    r = r.view(intervals, max_batch, n)
    a[:, live:] = float("nan")                            # idle rows may hold anything
    w4, outs = pack_int4(q), []
    for B in (max_batch, live):
        x, res = a[:, :B].contiguous(), r[:, :B].contiguous()
        out = torch.full((intervals, B, n), 7.0, dtype=torch.bfloat16, device=a.device)
        op = MatMulAddW4.new(x, w4, scales, res, out, intervals * B, n, k, group, zeros=z, max_batch=B)
        op.run(0, 1, live)
        torch.cuda.synchronize()
        outs.append(out[0, :live].clone())
        assert bool((out[0, live:] == 7.0).all()) and bool((out[1:] == 7.0).all())
        op.run(0, intervals, live)
        torch.cuda.synchronize()
        op.close()
        assert bool((out[:, live:] == 7.0).all())
        w = w4_weights(q, scales, z, group)
        ref, bound = a[:, :live].double() @ w.T, a[:, :live].double().abs() @ w.abs().T
        ref = ref + r[:, :live].double()
        # 1024 inputs of 64 product steps and 16 groups, at most four roundings of 2^-23 each: 4e-5; with more than 32 rows
        # in all the weights were rounded to bf16
        tol = HALF_BF16 * ref.abs() + 4e-5 * bound + (HALF_BF16 * bound if (intervals - 1) * B + live > 32 else 0.0)
        assert bool(((out[:, :live].double() - ref).abs() <= tol).all())
    assert torch.equal(*outs)                             # one interval: at most 32 rows, exact weights in both
