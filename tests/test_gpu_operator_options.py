"""What the options and the failure paths do to modified scores and a shared prefix: both ways a decode step can take its
prefix, waits that run out, steps on handles whose settings change, arguments that reach no kernel."""
import ctypes as C

import numpy as np
import pytest
import torch

from test_gpu_scores import Step as ScoreStep
from test_gpu_scores import windows
from test_gpu_shared_prefix import Step as PrefixStep

D = 128


# ------------------------------------------------------------------------------- a decode step's two ways through a prefix
@pytest.mark.gpu
@pytest.mark.parametrize("keys", [0, 1 << 40], ids=["tensor-memory", "split-KV"])
@pytest.mark.parametrize("heads", [(8, 1), (8, 8), (14, 2), (64, 1)], ids=str)
@pytest.mark.parametrize("shared,starts", [(1, [0]), (129, [-1, 70, 3]), (2050, list(range(0, 80, 4))), (777, [31] * 40)], ids=["1", "3", "20", "40"])
def test_both_kernels_take_any_prefix(keys, heads, shared, starts):
    s = PrefixStep(21, 1, starts, *heads, shared, max_batch=len(starts) + 1)
    op = s.op()
    op.set_option("prefix_flat_keys", keys)
    pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
    op.run_ragged(pos, 1, s.B)
    torch.cuda.synchronize()
    assert (op.kernel_stats()["prefill_tcgen05"][0] == 1) == (keys == 0)
    s.check()
    # back to back on the same workspace, queries changed in between
    s.q.mul_(-1.0)
    for _ in range(3):
        op.run_ragged(pos, 1, s.B)
    torch.cuda.synchronize()
    op.close()
    s.check()


@pytest.mark.gpu
@pytest.mark.parametrize("keys", [0, 1 << 40], ids=["tensor-memory", "split-KV"])
def test_repeated_steps_give_the_same_bits(keys):
    s = PrefixStep(22, 1, [5, 60, 200, 33] * 4, 16, 2, 5000)
    op = s.op()
    op.set_option("prefix_flat_keys", keys)
    pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
    outs = []
    for _ in range(6):
        op.run_ragged(pos, 1, s.B)
        torch.cuda.synchronize()
        outs.append((s.out.clone(), s.lse.clone()))
    op.close()
    assert all(torch.equal(o, outs[0][0]) and torch.equal(l, outs[0][1]) for o, l in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["scores", "prefix"])
def test_repeated_chunks_give_the_same_bits(form):
    if form == "scores":
        s = ScoreStep(23, 700, [0, 300], 16, 2, max_seq=1000).scores(30.0, True, begin=windows(2, 1000, 400))
    else:
        s = PrefixStep(23, 700, [0, 300], 16, 2, 1111)
    op = s.op()
    pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
    outs = []
    for _ in range(4):
        op.run_ragged(pos, 700, 2)
        torch.cuda.synchronize()
        outs.append((s.out.clone(), s.lse.clone()))
    op.close()
    assert all(torch.equal(o, outs[0][0]) and torch.equal(l, outs[0][1]) for o, l in outs)


# ------------------------------------------------------------------------------- waits that run out
@pytest.mark.gpu
@pytest.mark.parametrize("form,item", [("cap", 0), ("cap", 1), ("bias", 1), ("plain", 0), ("prefix", 1), ("prefix", 2), ("split", 0), ("split", 1)])
def test_a_tile_that_never_comes_is_reported_and_the_handle_goes_on(form, item):
    """The loader leaves one K or V tile unsignalled (nothing else is wrong), the wait on it runs out after 0.2 s, the
    kernel gives tensor memory back and returns, the run reports it, and the next run is right."""
    from ellm_b200 import EllmError
    from ellm_b200 import _lib as L
    if form in ("prefix", "split"):
        s = PrefixStep(24, 1 if form == "split" else 200, [0, 100, 31], 16, 2, 700)
    else:
        s = ScoreStep(24, 300, [0, 200], 16, 2, max_seq=520)
        s.scores(30.0 if form == "cap" else 0.0, form == "bias", begin=windows(2, 520, 200) if form == "plain" else None)
    op = s.op()
    op.set_option("prefix_flat_keys", 0)
    op.set_option("tc_wait_timeout_ns", 200_000_000)
    pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
    op.set_option("tc_debug_skip_kv_item", item)
    with pytest.raises(EllmError) as e:
        op.run_ragged(pos, s.rows, s.B)
    assert e.value.status == L.ERR_DEVICE_TIMEOUT
    op.set_option("tc_debug_skip_kv_item", -1)
    for _ in range(2):
        s.out.fill_(7.0)
        op.run_ragged(pos, s.rows, s.B)
        torch.cuda.synchronize()
        s.check()
    op.close()


# ------------------------------------------------------------------------------- caps outside the chunk kernel's range
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 150])
@pytest.mark.parametrize("cap", [0.05, 1.0, 128.0, 129.0, 1000.0, 1e6])
def test_caps_of_any_size(rows, cap):
    """Above 128 (and for a cap that is tiny against the scale) chunks take the warp-level kernel; the bar is the same
    up to cap 128 and beyond it the scores' error stays that of the fp32 product (the tanh's relative error near zero is
    2.5e-9, and |s| stays near 30 here)."""
    ScoreStep(25, rows, [0, 90], 8, 2, max_seq=260).scores(cap).run().check()


# ------------------------------------------------------------------------------- two streams, a long cache
@pytest.mark.gpu
def test_two_handles_on_two_streams_at_once():
    a = ScoreStep(26, 400, [0, 100], 16, 2, max_seq=520).scores(30.0, True)
    b = PrefixStep(26, 1, [10, 90, 40] * 5, 16, 2, 6000)
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    ops = [a.op(stream=st[0].cuda_stream, async_=True), b.op(stream=st[1].cuda_stream, async_=True)]
    ops[1].set_option("prefix_flat_keys", 0)
    pos = [torch.tensor(x.starts, dtype=torch.int32, device=x.dev) for x in (a, b)]
    torch.cuda.synchronize()
    for _ in range(20):
        ops[0].run_ragged(pos[0], 400, 2)
        ops[1].run_ragged(pos[1], 1, b.B)
    for op in ops:
        op.check()
    a.check()
    b.check()
    for op in ops:
        op.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 64])
def test_cache_offsets_past_32_bits(rows):
    """Sequence slots 2^31 elements apart: offsets pass 32 bits in elements, 33 in bytes."""
    from ellm_b200 import Attention
    dev = torch.device("cuda:0")
    big = torch.empty((2 << 31) + (1 << 20), dtype=torch.bfloat16, device=dev)   # 8.6 GB, touched where it is used
    L, H, Hkv = 300, 8, 2
    s = ScoreStep(27, rows, [40, 200], H, Hkv, max_seq=L).scores(30.0, True, begin=windows(2, L, 100))
    strides = (1 << 31, L * D, D, 1)
    views = []
    for at, src in ((0, s.k), (1 << 19, s.v)):
        t = torch.as_strided(big, (2, Hkv, L, D), strides, at)
        t.copy_(src)
        views.append(t)
    s.k, s.v = views
    s.strides = list(strides)
    s.run().check()
    pre = PrefixStep(27, rows, [40, 200], H, Hkv, 500)
    far = torch.as_strided(big, (Hkv, 505, D), (1 << 31, D, 1), 1 << 18)
    far.copy_(pre.pk)
    pre.pk = far
    far_v = torch.as_strided(big, (Hkv, 505, D), (1 << 31, D, 1), (1 << 18) + 505 * D)
    far_v.copy_(pre.pv)
    pre.pv = far_v
    pre.run().check()


# ------------------------------------------------------------------------------- arguments (no GPU needed)
def test_null_handles_are_refused():
    import ellm_b200
    from ellm_b200 import _lib as L
    lib = ellm_b200.load()
    scores = L.AttnScores(1.0, None, None, 0, None)
    assert lib.ellm_attn_set_scores(None, C.byref(scores)) == L.ERR_INVALID_ARG
    assert lib.ellm_attn_set_shared_prefix(None, 0x1000, 0x1000, 128, 128, 4) == L.ERR_INVALID_ARG
    assert lib.ellm_matmul_add_w4_run(None, 0, 1, 1, 1, 0) == L.ERR_INVALID_ARG
    assert lib.ellm_matmul_add_w4_create(None, None) == L.ERR_INVALID_ARG
    assert lib.ellm_matmul_add_w4_destroy(None) == L.OK


def test_tensors_of_another_place_or_type_are_refused():
    """The Python mirror's own checks, ahead of any call into the library."""
    from ellm_b200 import Attention, MatMulAddW4
    from ellm_b200 import _lib as L
    op = object.__new__(Attention)
    op._h, op.desc = None, L.AttnDesc()
    op.desc.q_heads, op.desc.kv_heads, op.desc.head_size, op.desc.max_batch, op.desc.max_seq = 8, 2, D, 3, 40
    for kw in (dict(slopes=torch.zeros(8)), dict(prefix_lens=torch.zeros(3, dtype=torch.int32)),
               dict(row_begin=torch.zeros(3, 40, dtype=torch.int32)), dict(row_begin=torch.zeros(3, 40)),
               dict(row_begin=torch.zeros(3, 39, dtype=torch.int32))):
        with pytest.raises(ValueError):
            op.set_scores(1.0, **kw)
    kv = torch.zeros(2, 9, D, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        op.set_shared_prefix(kv, kv)
    with pytest.raises(ValueError):
        MatMulAddW4.new(0x1000, torch.zeros(8, 64, dtype=torch.uint8), 0x1000, None, 0x1000, 1, 8, 128, 32)
