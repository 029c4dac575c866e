"""What a capped row's result depends on: the products of masked keys, and of the lanes of a row tile that hold no row, have no
part in which form of the tanh its warp takes (the forms differ by 1e-7 of the cap, enough to turn a rounding to bf16)."""
import numpy as np
import pytest
import torch

from test_gpu_scores import Step, windows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap,bias", [(50.0, False), (20.0, True), (100.0, False)])
@pytest.mark.parametrize("heads", [(15, 3), (16, 2), (60, 3)], ids=str)
@pytest.mark.parametrize("mask", ["causal", "window"])
def test_finite_masked_keys_change_no_bit(cap, bias, heads, mask):
    """Keys that no row sees: small ones, then ones whose products lie far beyond the cap."""
    rows, start, L = 140, 100, 400
    s = Step(141, rows, [start], *heads, L, sharp=1.0)
    begin = windows(1, L, 70) if mask == "window" else None
    s.scores(cap, bias, begin)
    seen = slice(start - 69 if mask == "window" else 0, start + rows)
    outs = []
    for f in (0.0, 1.0, 300.0):
        k, v = torch.randn(2, 1, heads[1], L, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(s.dev) * f
        k[:, :, seen], v[:, :, seen] = s.k[:, :, seen], s.v[:, :, seen]
        s.k, s.v = k, v
        s.strides = [k.stride(i) for i in range(4)]
        s.out.fill_(7.0)
        s.run(1 if 128 % (heads[0] // heads[1]) == 0 else 0, ragged=True)
        outs.append((s.out.clone(), s.lse.clone()))
    s.check()
    assert all(torch.equal(o, outs[0][0]) and torch.equal(l, outs[0][1]) for o, l in outs)


@pytest.mark.parametrize("cap,bias", [(50.0, False), (20.0, True), (100.0, False)])
@pytest.mark.parametrize("heads", [(15, 3), (60, 3), (14, 2)], ids=str)
def test_lanes_without_a_row_change_no_bit(cap, bias, heads):
    """Groups that do not fill a row tile, between runs of another operator whose queries are huge or small: its tiles are
    what the unused part of shared memory holds."""
    s = Step(142, 129, [int(x) for x in np.random.default_rng(1).integers(0, 130, 20)], *heads, 290).scores(cap, bias)
    fill = Step(143, 300, [0, 0, 0], 64, 8, 300, sharp=1.0).scores(30.0)
    pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
    op, other = s.op(), fill.op()
    outs = []
    for f in (1e-3, 1.0, 1e4, 1e-3, 1e4):
        fill.q.copy_((torch.randn(fill.q.shape, generator=torch.Generator().manual_seed(4)) * f).to(torch.bfloat16))
        for _ in range(3):
            other.run(0, 300, 3)
            op.run_ragged(pos, 129, s.B)
            outs.append((s.out.clone(), s.lse.clone()))
    torch.cuda.synchronize()
    op.close()
    other.close()
    s.check()
    assert all(torch.equal(o, outs[0][0]) and torch.equal(l, outs[0][1]) for o, l in outs)
