"""A row's unnormalised weights are rounded to bf16 once, also where a maximum leaps between the two halves of a key tile: the
first half's weights, stored already, are brought to the new maximum by a power of two.  Keys of one tile of which one in its
first half lies 15 powers of two above all keys before it and one in its second half 16, so that the step goes on past the
first and rescales at the second; V holds a channel for each, so that the outputs are the two weights themselves.

The bar of operator_refs: 2^-8 for the weight, 2^-8 for the result, 1e-3 for the score.  A second rounding of the weight
passes it in some 0.6 % of rows whose mantissas are near 1 (three roundings of up to 2^-8)."""
import numpy as np
import pytest
import torch

from operator_refs import assert_attention, attention_ref

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("kind", ["scores", "capped", "prefix"])
@pytest.mark.parametrize("order", [1, 2])
def test_weights_of_a_tile_in_which_the_maximum_leaps(kind, order):
    from ellm_b200 import Attention
    dev, H, rows, L = torch.device("cuda:0"), 16, 600, 1000
    g = torch.Generator().manual_seed(151)
    q = torch.zeros(rows, 1, H, D)
    q[..., :32] = 4.0 * (1.0 + 0.01 * torch.randn(rows, 1, H, 32, generator=g))
    q = q.to(torch.bfloat16).to(dev)
    k, v = torch.zeros(2, 1, 1, L, D, dtype=torch.bfloat16, device=dev)
    first, second = 128 * order + 10, 128 * order + 70
    k[0, 0, first, :16], k[0, 0, second, 16:32] = 1.84375, 1.9765625     # 15.05 and 16.13 in powers of two
    v[0, 0, first, 0] = v[0, 0, second, 1] = 1.0
    out, lse = torch.zeros_like(q), torch.zeros(rows, 1, H, device=dev)
    P = 384 if kind == "prefix" else 0
    own_k, own_v = k[:, :, P:].contiguous(), v[:, :, P:].contiguous()
    start = L - rows - P
    op = Attention.new(q, own_k, own_v, out, 1, H, 1, D, [own_k.stride(i) for i in range(4)], D ** -0.5, max_seq=L - P, max_interval=rows,
                       lse=lse, prefill_kernel=1)
    cap = 100.0 if kind == "capped" else 0.0
    if P:
        op.set_shared_prefix(k[0, :, :P], v[0, :, :P])
    else:
        op.set_scores(cap, row_begin=torch.zeros(1, L, dtype=torch.int32, device=dev))
    op.run(start, rows, 1)
    torch.cuda.synchronize()
    op.close()
    pos = P + start + np.arange(rows)
    ref, A, want = attention_ref(q[:, 0], k[0], v[0], np.zeros_like(pos), pos + 1, pos, D ** -0.5, cap)
    assert 0.2 < ref[..., 0].min().item() and ref[..., 1].max().item() < 0.8       # both weights count
    assert_attention(out[:, 0], ref, A, lse[:, 0], want)
