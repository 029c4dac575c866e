"""Rows that the chunk kernels compute once more, key by key, because the tiles they were computed from hold NaN or infinity
(Attention.set_scores, Attention.set_shared_prefix): the second result is the one that stays, and the time it takes counts
against no device-side wait."""
import numpy as np
import pytest
import torch

from operator_refs import HALF_BF16, assert_attention, attention_ref
from test_gpu_scores import Step as ScoreStep
from test_gpu_shared_prefix import Step as PrefixStep

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("kernel", [1, 2])
def test_recomputed_rows_replace_the_first_result_in_every_run(kernel):
    """Masked keys that are NaN in the tiles of most rows; outputs and LSE of repeated runs over poisoned buffers."""
    s = ScoreStep(41, 300, [0], 8, 1, max_seq=300)
    begin = np.zeros((1, 300), dtype=np.int32)
    begin[0, 60:] = 60
    s.scores(20.0, True, begin=begin)
    s.k[0, :, 10:50] = float("nan")
    s.v[0, :, 10:50] = float("nan")
    op = s.op(kernel)
    pos, lo, hi = s.intervals(0)
    ref, A, lse = attention_ref(s.q[:, 0], s.k[0], torch.nan_to_num(s.v[0], 0.0, 0.0, 0.0), lo, hi, pos, D ** -0.5, 20.0, s.slopes)
    first = None
    for _ in range(20):
        s.out.fill_(float("nan"))
        s.lse.fill_(float("nan"))
        op.run(0, 300, 1)
        got = s.out[60:, 0].clone(), s.lse[60:, 0].clone()
        first = first or got
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
    assert_attention(first[0], ref[60:], A[60:], first[1], lse[60:])
    op.close()


def check_but_one_column(out, ref, A, lse, lse_ref):
    """Column 0 is infinite in every row; the others are held to the usual bar."""
    assert bool(torch.isposinf(out[..., 0]).all())
    got, r, a = out[..., 1:].double(), ref[..., 1:], A[..., 1:]
    assert ((got - r).abs() / ((HALF_BF16 + 1e-3) * a + HALF_BF16 * r.abs() + 1e-6)).max().item() <= 1.0
    assert (lse.double() - lse_ref).abs().max().item() <= 1e-3


@pytest.mark.parametrize("kind", ["scores", "prefix"])
def test_the_time_of_recomputed_rows_counts_against_no_wait(kind):
    """One visible V value is infinite, so that every row is computed twice, the second time by one warp over some thousand
    keys (tens of milliseconds a warp); there are 160 items, more than SMs, so that other warps have work to wait for, and every
    wait is limited to 5 ms."""
    rows, history, H, Hkv, B = 160, 12000, 64, 8, 4
    if kind == "scores":
        s = ScoreStep(42, rows, [history] * B, H, Hkv, max_seq=history + rows, sharp=0.5).scores(20.0)
        s.v[:, :, 7, 0] = float("inf")
    else:
        s = PrefixStep(42, rows, [0] * B, H, Hkv, history, sharp=0.5)
        s.pv[:, 7, 0] = float("inf")
    op = s.op()
    op.set_option("tc_wait_timeout_ns", 5_000_000)
    op.run(s.starts[0], rows, B)
    assert op.kernel_stats()["prefill_tcgen05"][0] == 1
    op.close()
    at = torch.tensor([0, 1, 77, rows - 1], device=s.dev)          # (the reference of a few rows)
    for b in range(B):
        pos = s.starts[b] + at.cpu().numpy()
        if kind == "scores":
            ref = attention_ref(s.q[at, b], s.k[b], s.v[b], np.zeros_like(pos), pos + 1, pos, D ** -0.5, 20.0)
        else:
            k, v = (torch.cat((p[:, :s.P], own[b, :, :rows]), 1) for p, own in ((s.pk, s.k), (s.pv, s.v)))
            ref = attention_ref(s.q[at, b], k, v, np.zeros_like(pos), pos + 1 + s.P, pos, D ** -0.5, shared=s.P)
        check_but_one_column(s.out[at, b], ref[0], ref[1], s.lse[at, b], ref[2])
