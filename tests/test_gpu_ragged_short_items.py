"""Ragged chunks of many short items: more items than SMs, each of one or two key tiles that end inside a tile, so that the
loader is done with the next item while the products still wait for this one's last.  Plain attention, modified scores and a
shared prefix, many runs of each; every run gives the same bits, and the first is held against the 64-bit reference.

The model below is the order of events behind the faulty form of this: a barrier's phase tells one completion from two only
if the waiter has seen the first."""
import numpy as np
import pytest
import torch

from operator_refs import assert_attention, attention_ref
from test_gpu_scores import Step as ScoreStep
from test_gpu_scores import documents, windows
from test_gpu_shared_prefix import Step as PrefixStep

D = 128
RUNS = 150


class Barrier:
    def __init__(self):
        self.phase = 0

    def arrive(self):
        self.phase += 1

    def passed(self, parity):
        return self.phase % 2 != parity


def test_a_barrier_that_completes_twice_before_it_is_looked_at_looks_untouched():
    """One barrier for the clean-ups of two items against one per ring slot, in the order that stalls the former."""
    one = Barrier()
    one.arrive()                        # item n cleaned up, the products of its last step not yet due
    assert one.passed(0)
    one.arrive()                        # item n + 1, of two tiles, cleaned up as well
    assert not one.passed(0)            # item n's products would wait for good
    slots = [Barrier() for _ in range(5)]
    slots[3].arrive()                   # item n's last V tile; its slot is refilled only once the products have used it
    for s in (4, 0):
        slots[s].arrive()
    assert slots[3].passed(0) and slots[4].passed(0) and slots[0].passed(0)


def repeat(op, pos, s):
    first = None
    for i in range(RUNS):
        op.run_ragged(pos, s.rows, s.B)
        torch.cuda.synchronize()
        if i % 10 == 0:
            got = s.out.clone(), s.lse.clone()
            first = first or got
            assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])


SHAPES = [(64, 9, 60, 3), (129, 20, 15, 3), (5, 40, 80, 4), (100, 40, 12, 1), (100, 9, 64, 1), (40, 30, 32, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,B,H,Hkv", SHAPES, ids=str)
@pytest.mark.parametrize("cap,bias,mask", [(50.0, False, None), (0.0, True, "documents"), (100.0, True, "window"), (0.0, False, "window")])
def test_scores(rows, B, H, Hkv, cap, bias, mask):
    rng = np.random.default_rng(rows + B)
    starts = [int(x) for x in rng.integers(0, 150, B)]
    max_seq = max(starts) + rows + 20
    begin = {None: None, "documents": documents(3, B, max_seq, 40), "window": windows(B, max_seq, 60)}[mask]
    s = ScoreStep(131, rows, starts, H, Hkv, max_seq).scores(cap, bias, begin)
    op = s.op()
    repeat(op, torch.tensor(starts, dtype=torch.int32, device=s.dev), s)
    op.close()
    s.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,B,H,Hkv", SHAPES, ids=str)
def test_shared_prefix(rows, B, H, Hkv):
    rng = np.random.default_rng(rows + B + 1)
    s = PrefixStep(132, rows, [int(x) for x in rng.integers(0, 5, B)], H, Hkv, 1)
    op = s.op()
    repeat(op, torch.tensor(s.starts, dtype=torch.int32, device=s.dev), s)
    op.close()
    s.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,B,H,Hkv", [(64, 20, 64, 4), (128, 40, 16, 4), (100, 40, 32, 1), (100, 9, 64, 1), (40, 30, 32, 8)], ids=str)
def test_plain_attention(rows, B, H, Hkv):
    from ellm_b200 import Attention
    rng = np.random.default_rng(rows + B + 2)
    starts = [int(x) for x in rng.integers(0, 150, B)]
    s = ScoreStep(133, rows, starts, H, Hkv, max(starts) + rows + 20)
    op = Attention.new(s.q, s.k, s.v, s.out, s.mb, H, Hkv, D, s.strides, D ** -0.5, max_seq=s.max_seq, max_interval=rows, lse=s.lse,
                       prefill_kernel=1)
    repeat(op, torch.tensor(starts, dtype=torch.int32, device=s.dev), s)
    op.close()
    for b in range(B):
        pos = starts[b] + np.arange(rows)
        ref, A, lse = attention_ref(s.q[:, b], s.k[b], s.v[b], np.zeros_like(pos), pos + 1, pos, D ** -0.5)
        assert_attention(s.out[:, b], ref, A, s.lse[:, b], lse)
