"""MatMulAddW4's launches: they are timed when profiling is on, and their waits do not count the time of the kernel before."""
import numpy as np
import pytest
import torch

from operator_refs import assert_w4, w4_weights
from test_gpu_w4 import make

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("rows,kernel,launches", [(5, 0, 1), (5, 1, 2), (80, -1, 2)], ids=["warp", "tensor-memory", "many"])
def test_profiling_times_every_run(rows, kernel, launches):
    """1152 x 1024 is 9 tiles of 8 blocks on 148 SMs at most: every tile is cut, a run is two launches on that kernel."""
    from ellm_b200 import MatMulAddW4, pack_int4
    q, scales, z, a, r = make(61, rows, 1152, 1024, 64, True, True)
    out = torch.zeros(rows, 1152, dtype=torch.bfloat16, device=a.device)
    op = MatMulAddW4.new(a, pack_int4(q), scales, r, out, rows, 1152, 1024, 64, zeros=z)
    op.set_pairing(kernel)
    op.run(0, 1, rows)
    assert op.kernel_stats() == (launches, 0, 0.0)
    op.set_profiling(True)
    for _ in range(3):
        op.run(0, 1, rows)
    torch.cuda.synchronize()
    n, timed, ms = op.kernel_stats()
    assert n == 4 * launches and timed == 3 and 3e-3 < ms < 30.0
    op.set_profiling(False)
    op.run(0, 1, rows)
    torch.cuda.synchronize()
    assert op.kernel_stats()[1:] == (timed, ms)
    assert_w4(out, a, w4_weights(q, scales, z, 64), r, rows > 32)
    op.close()


@pytest.mark.parametrize("rows", [16, 200])
def test_the_time_of_the_kernel_before_counts_against_no_wait(rows):
    """A chunk of few rows over a long history keeps a few SMs busy for some milliseconds; the projection behind it starts
    early on the others and waits there, and every wait of its own is limited to 0.3 ms."""
    from ellm_b200 import Attention, MatMulAddW4, pack_int4
    dev, H, Hkv, L, chunk = torch.device("cuda:0"), 16, 1, 150_000, 32
    g = torch.Generator(device=dev).manual_seed(62)
    q_att = torch.randn(chunk, 1, H, D, generator=g, device=dev).to(torch.bfloat16)
    kv = torch.randn(2, 1, Hkv, L, D, generator=g, device=dev).to(torch.bfloat16)
    att = torch.zeros_like(q_att)
    q, scales, z, a, r = make(62, rows, 2048, 2048, 64, True, True)
    out = torch.zeros(rows, 2048, dtype=torch.bfloat16, device=dev)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    attn = Attention.new(q_att, kv[0], kv[1], att, 1, H, Hkv, D, [kv[0].stride(i) for i in range(4)], D ** -0.5, max_seq=L,
                         max_interval=chunk, prefill_kernel=1, stream=stream.cuda_stream, async_=True)
    op = MatMulAddW4.new(a, pack_int4(q), scales, r, out, rows, 2048, 2048, 64, zeros=z, stream=stream.cuda_stream, async_=True)
    op.set_pairing(1)
    torch.cuda.synchronize()
    op.set_wait_timeout(300_000)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(3):
        with torch.cuda.stream(stream):
            start.record()
            attn.run(L - chunk, chunk, 1)
            op.run(0, 1, rows)
            end.record()
        op.check()
        attn.check()
    assert start.elapsed_time(end) > 0.6              # the chunk alone is well past the limit
    assert_w4(out, a, w4_weights(q, scales, z, 64), r, rows > 32)
    for o in (attn, op):
        o.close()
