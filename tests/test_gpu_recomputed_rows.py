"""Rows that the chunk kernels compute once more, key by key, because the tiles they were computed from hold NaN or infinity
(Attention.set_scores): the second result is the one that stays."""
import numpy as np
import pytest
import torch

from operator_refs import assert_attention, attention_ref
from test_gpu_scores import Step as ScoreStep

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
