"""Tensors given to set_scores and set_shared_prefix that are replaced while steps that read them are still queued on the
operator's stream, another one than the tensors' own: their memory is not handed out again before those steps are done."""
import pytest
import torch

from test_gpu_scores import Step as ScoreStep
from test_gpu_scores import windows
from test_gpu_shared_prefix import Step as PrefixStep

D = 128


def busy(stream, ms):
    """Work of a few milliseconds ahead of the steps."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(int(ms * 2e6))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 200])
def test_scores(rows):
    s = ScoreStep(101, rows, [40, 300], 16, 2, max_seq=520).scores(30.0, True, begin=windows(2, 520, 90))
    stream = torch.cuda.Stream()
    pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
    op = s.op(stream=stream.cuda_stream, async_=True)
    slopes, begin = s.slopes.clone(), s.begin.clone()          # (what the check reads)
    op.run_ragged(pos, rows, 2)
    torch.cuda.synchronize()
    s.out.fill_(7.0)
    torch.cuda.synchronize()
    busy(stream, 20)
    op.run_ragged(pos, rows, 2)
    op.set_scores(5.0)                                         # the operator lets go of the tensors, and so does this test
    s.slopes, s.begin = slopes, begin
    spoil = [torch.full_like(t, 1000) for _ in range(40) for t in (slopes, begin)]
    torch.cuda.current_stream().synchronize()
    op.check()
    s.check()
    op.close()
    del spoil


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("keys", [0, 1 << 40])
def test_prefix(rows, keys):
    s = PrefixStep(102, rows, [40, 10], 16, 2, 900)
    stream = torch.cuda.Stream()
    pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
    pk, pv = s.pk.clone(), s.pv.clone()
    s.pk, s.pv = s.pk.clone(), s.pv.clone()                    # (tensors of their own, not views that others hold)
    op = s.op(stream=stream.cuda_stream, async_=True)
    op.set_option("prefix_flat_keys", keys)
    op.run_ragged(pos, rows, 2)
    torch.cuda.synchronize()
    busy(stream, 20)
    op.run_ragged(pos, rows, 2)
    op.set_shared_prefix(None, None)
    s.pk, s.pv = pk, pv
    spoil = [torch.full_like(pk, 50.0) for _ in range(20)]
    torch.cuda.current_stream().synchronize()
    op.check()
    s.check()
    op.close()
    del spoil
