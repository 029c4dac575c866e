"""Projections with 4-bit weights (MatMulAddW4) against a 64-bit reference: every group size, rows from one to a
prompt chunk, odd column counts, strides, idle rows."""
import pytest
import torch

from operator_refs import assert_w4, w4_weights

D = 128


def make(seed, rows, n, k, group, zeros, residual, max_batch=None, dev="cuda:0", pad=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = ((torch.rand(n, k // group, generator=g) + 0.1) * 0.05).to(torch.bfloat16)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    a = torch.randn(rows, k + pad, generator=g).to(torch.bfloat16)
    r = torch.randn(rows, n + pad, generator=g).to(torch.bfloat16) if residual else None
    return [t.to(dev) if t is not None else None for t in (q, scales, z, a, r)]


def run(seed, rows, n, k, group, zeros=True, residual=True, pad=0, live=None, chunk=False, kernel=-1):
    from ellm_b200 import MatMulAddW4, pack_int4
    q, scales, z, a, r = make(seed, rows, n, k, group, zeros, residual, pad=pad)
    out = torch.full((rows, n + pad), 7.0, dtype=torch.bfloat16, device=a.device)
    op = MatMulAddW4.new(a, pack_int4(q), scales, r, out, rows, n, k, group, zeros=z, a_row_stride=k + pad,
                         residual_row_stride=n + pad, output_row_stride=n + pad, max_batch=1 if chunk else rows)
    op.set_pairing(kernel)
    live = rows if live is None else live
    op.run(0, *((live, 1) if chunk else (1, live)))
    torch.cuda.synchronize()
    op.close()
    w = w4_weights(q, scales, z, group)
    assert_w4(out[:live, :n], a[:live, :k], w, r[:live, :n] if residual else None, rounded_weights=live > 32 or (rows > 32 and not chunk))
    assert bool((out[live:] == 7.0).all()) and bool((out[:, n:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16])
@pytest.mark.parametrize("zeros,residual", [(False, False), (True, True)])
@pytest.mark.parametrize("kernel", [0, 1])
def test_few_rows(group, rows, zeros, residual, kernel):
    run(1, rows, 264, 1024, group, zeros, residual, kernel=kernel)


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(8, 128), (16, 256), (40, 384), (2368, 640), (4744, 512), (5120, 2048), (9480, 1152), (30000, 256)], ids=str)
@pytest.mark.parametrize("rows", [1, 13])
@pytest.mark.parametrize("kernel", [0, 1])
def test_few_rows_sizes(n, k, rows, kernel):
    run(2, rows, n, k, 64 if k % 256 else 32, kernel=kernel)
    run(3, rows, n, k, 128, zeros=False, residual=False, kernel=kernel)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [17, 32, 33, 100, 256, 257, 300, 700])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_many_rows(rows, group):
    run(4, rows, 520, 768, group, chunk=True)
    run(5, rows, 256, 384, group, zeros=False, residual=False)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [16, 40, 513])
@pytest.mark.parametrize("n,k", [(8, 128), (128, 128), (19000, 128), (136, 8192), (9480, 640)], ids=str)
def test_tiles_cut_between_ctas(rows, n, k):
    run(6, rows, n, k, 128, kernel=1, chunk=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 16, 40])
@pytest.mark.parametrize("kernel", [0, 1])
def test_strides_and_idle_rows(rows, kernel):
    run(6, rows, 136, 256, 64, pad=24, kernel=kernel)
    run(7, rows, 136, 256, 64, live=rows - 3, kernel=kernel)
    run(8, rows, 136, 256, 64, live=rows - 3, chunk=True, kernel=kernel)


@pytest.mark.gpu
@pytest.mark.parametrize("kernel", [0, 1])
def test_extreme_weights_are_exact(kernel):
    """All 16 numbers, zero points 0 and 15, one-hot rows: the products come out as (q - z) * scale rounded once."""
    from ellm_b200 import MatMulAddW4, pack_int4
    dev = "cuda:0"
    n, k = 32, 128
    q = (torch.arange(n)[:, None] + torch.arange(k)[None]).remainder(16).to(torch.uint8).to(dev)
    scales = torch.full((n, 4), 3.0, dtype=torch.bfloat16, device=dev)
    z = torch.tensor([0, 15, 8, 127], dtype=torch.uint8, device=dev).repeat(n, 1)
    for i0 in range(0, k, 16):
        a = torch.zeros(16, k, dtype=torch.bfloat16, device=dev)
        a[torch.arange(16), i0 + torch.arange(16)] = 1.0
        out = torch.zeros(16, n, dtype=torch.bfloat16, device=dev)
        op = MatMulAddW4.new(a, pack_int4(q), scales, None, out, 16, n, k, 32, zeros=z)
        op.set_pairing(kernel)
        op.run(0, 1, 16)
        torch.cuda.synchronize()
        op.close()
        want = ((q.float() - z.float().repeat_interleave(32, 1)) * 3.0)[:, i0:i0 + 16].T.to(torch.bfloat16)
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kernel", [0, 1])
def test_results_do_not_depend_on_timing_and_the_output_may_be_the_residual(kernel):
    from ellm_b200 import MatMulAddW4, pack_int4
    q, scales, z, a, r = make(9, 11, 1032, 4096, 64, True, True)
    w4 = pack_int4(q)
    outs = []
    for _ in range(5):
        y = r.clone()
        op = MatMulAddW4.new(a, w4, scales, y, y, 11, 1032, 4096, 64, zeros=z)
        op.set_pairing(kernel)
        op.run(0, 1, 11)
        torch.cuda.synchronize()
        op.close()
        outs.append(y)
    assert all(torch.equal(outs[0], y) for y in outs[1:])
    assert_w4(outs[0], a, w4_weights(q, scales, z, 64), r, False)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 64])
def test_captured_and_replayed_with_new_inputs_and_weights(rows):
    from ellm_b200 import MatMulAddW4, pack_int4
    q, scales, z, a, r = make(10, rows, 512, 1024, 128, True, True)
    w4, out = pack_int4(q), torch.zeros(rows, 512, dtype=torch.bfloat16, device="cuda:0")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        op = MatMulAddW4.new(a, w4, scales, r, out, rows, 512, 1024, 128, zeros=z, stream=stream.cuda_stream, async_=True)
        op.run(0, 1, rows)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            op.run(0, 1, rows)
        a.mul_(0.5)
        q = (15 - q)
        w4.copy_(pack_int4(q))
        graph.replay()
        stream.synchronize()
    assert_w4(out, a, w4_weights(q, scales, z, 128), r, rows > 32)
    op.check()
    del graph
    op.close()


def test_refusals():
    from ellm_b200 import EllmError, MatMulAddW4, pack_int4
    P = 0x10000

    def new(**kw):
        args = dict(ptr1=P, w4_ptr=P, scales_ptr=P, ptr3=None, output_ptr=P, m_max=4, n_max=64, k_max=256, group=64)
        args.update(kw)
        return MatMulAddW4.new(**args)
    for kw in (dict(ptr1=None), dict(w4_ptr=None), dict(scales_ptr=None), dict(output_ptr=None), dict(group=16), dict(group=256),
               dict(group=0), dict(k_max=192), dict(k_max=0), dict(n_max=12), dict(n_max=0), dict(m_max=0), dict(m_max=4, max_batch=3),
               dict(ptr1=P + 2), dict(w4_ptr=P + 4), dict(zeros=P + 1), dict(a_row_stride=100), dict(output_row_stride=32)):
        with pytest.raises(EllmError):
            new(**kw)
    with pytest.raises(ValueError):
        pack_int4(torch.zeros(4, 3, dtype=torch.uint8))
    with pytest.raises(ValueError):
        pack_int4(torch.zeros(4, 4))
    w = torch.zeros(64, 128, dtype=torch.uint8)
    with pytest.raises(ValueError):                        # not on the GPU
        new(w4_ptr=w)
    assert pack_int4(torch.tensor([[1, 2, 15, 0]], dtype=torch.uint8)).tolist() == [[0x21, 0x0F]]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [16, 80])
def test_a_load_that_never_comes_is_reported_and_the_handle_goes_on(rows):
    from ellm_b200 import EllmError, MatMulAddW4, pack_int4
    from ellm_b200 import _lib as L
    q, scales, z, a, r = make(12, rows, 256, 1024, 128, True, True)
    out = torch.zeros(rows, 256, dtype=torch.bfloat16, device="cuda:0")
    op = MatMulAddW4.new(a, pack_int4(q), scales, r, out, rows, 256, 1024, 128, zeros=z)
    op.set_pairing(1)
    op.set_wait_timeout(20_000_000)
    op.debug_skip_load(0)
    with pytest.raises(EllmError) as e:
        op.run(0, 1, rows)
    assert e.value.status == L.ERR_DEVICE_TIMEOUT
    op.debug_skip_load(-1)
    op.run(0, 1, rows)
    torch.cuda.synchronize()
    assert_w4(out, a, w4_weights(q, scales, z, 128), r, rows > 32)
    op.close()


@pytest.mark.gpu
def test_run_refusals():
    from ellm_b200 import EllmError, MatMulAddW4, pack_int4
    q, scales, z, a, _ = make(11, 8, 64, 128, 32, True, False)
    out = torch.full((8, 64), 7.0, dtype=torch.bfloat16, device="cuda:0")
    op = MatMulAddW4.new(a, pack_int4(q), scales, None, out, 8, 64, 128, 32, zeros=z, max_batch=4)
    for bad in ((0, 3, 1), (0, 1, 5), (0, 1 << 62, 1)):
        with pytest.raises(EllmError):
            op.run(*bad)
    op.run(0, 0, 4)
    op.run(0, 2, 0)
    op.run(0, 1, 4, 2, 1)                                  # another thread id launches nothing
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())
    op.close()
