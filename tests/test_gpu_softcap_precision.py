"""The capped score itself.  A row that sees one key has an LSE of exactly that key's score, cap * tanh(scale * q.k / cap), so
the LSE shows the tanh without a softmax around it.  Queries and keys are small whole numbers: products and sums are exact
and the only errors are those of the score's own arithmetic:

  tanh: the polynomial up to |u| = 1 is off by 6.1e-7 of its value, the exponential form by 1e-7 absolute (3e-7 with the
  roundings of its argument and of the fast exponential), either by less than 6e-7 of cap; its multiply-adds, the products
  with cap and log2(e), the subtraction of the maximum and the way back to natural units are at most 16 roundings of 2^-24 of
  at most cap: (6e-7 + 16 * 2^-24) cap = 1.6e-6 cap; the weight itself, exp2 of about 0, adds 2^-22 to the logarithm.
  A bias (slope 1/4, a key's distance to itself is 0) is taken off and put back at up to 46 in log2 units: two roundings
  of 2^-19."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


def run(cap, rows, kernel, top, bias=False):
    """Row r's own key gives the product t[r]; every product of the chunk is within `top` caps.  Returns LSE and scores."""
    from ellm_b200 import Attention
    dev, H, scale = torch.device("cuda:0"), 8, D ** -0.5
    n = max(rows, 256)
    t = np.round(np.linspace(0.0, top * cap / scale, n)) * np.where(np.arange(n) % 3 == 0, -1.0, 1.0)
    keys = torch.zeros(n, D, dtype=torch.float64)
    for r in range(n):                       # whole numbers of one sign, of at most 8 bits, that add up to t[r]
        base, rest = divmod(int(abs(t[r])), D)
        keys[r] = base
        keys[r, :rest] += 1
        keys[r] *= np.sign(t[r]) if t[r] else 1.0
    assert keys.abs().max() <= 255
    k = keys.to(torch.bfloat16).to(dev).view(1, 1, n, D).contiguous()
    assert torch.equal(k.double().cpu().view(n, D), keys)
    v = torch.ones_like(k)
    q = torch.ones(rows, 1, H, D, dtype=torch.bfloat16, device=dev)
    out, lse = torch.zeros_like(q), torch.zeros(rows, 1, H, device=dev)
    op = Attention.new(q, k, v, out, 1, H, 1, D, [k.stride(i) for i in range(4)], scale, max_seq=n, max_interval=rows, lse=lse,
                       prefill_kernel=kernel)
    slopes = torch.full((H,), 0.25, device=dev) if bias else None       # (a key's distance to itself is 0)
    op.set_scores(cap, slopes, torch.arange(n, dtype=torch.int32, device=dev)[None].contiguous())
    got = []
    if rows == 1:
        for p in range(0, n, 5):
            op.run(p, 1, 1)
            got.append(lse[0, 0].cpu().double().numpy())
        t = t[::5]
    else:
        op.run(0, rows, 1)
        got = lse[:, 0].cpu().double().numpy()
    torch.cuda.synchronize()
    assert (op.kernel_stats()["prefill_tcgen05"][0] > 0) == (rows > 1 and kernel == 1)
    op.close()
    return np.asarray(got), t * scale


@pytest.mark.parametrize("rows,kernel", [(256, 1), (700, 1), (256, 2), (1, 0)], ids=["chunk", "long chunk", "warp-level", "step"])
@pytest.mark.parametrize("cap", [5.0, 30.0, 50.0, 61.0, 62.0, 100.0, 128.0])
@pytest.mark.parametrize("top", [0.24, 0.99, 2.5])
@pytest.mark.parametrize("bias", [False, True])
def test_the_capped_score(rows, kernel, cap, top, bias):
    lse, s = run(cap, rows, kernel, top, bias)
    err = np.abs(lse - (cap * np.tanh(s / cap))[:, None])
    assert err.max() <= 1.6e-6 * cap + 2.0 ** -22 + (2.0 ** -18 if bias else 0.0), f"{err.max():.3g} at cap {cap}"


@pytest.mark.parametrize("cap", [62.0, 100.0, 128.0])
@pytest.mark.parametrize("bias", [False, True])
def test_large_caps_at_the_top_of_the_polynomials_range(cap, bias):
    """Many keys with scores up to the cap, a running maximum that moves: against the 64-bit reference."""
    from test_gpu_scores import Step
    s = Step(81, 300, [0, 130], 16, 2, max_seq=440, sharp=1.0).scores(cap, bias)
    top = max((torch.einsum("rhd,kd->rhk", s.q[:, b].float(), torch.nan_to_num(s.k[b, 0].float())).abs().max().item()) for b in range(2))
    s.q.copy_((s.q.float() * (0.97 * cap / (top * D ** -0.5))).to(torch.bfloat16))
    s.run(1).check()
    s.run(2).check()
