"""Decode steps that take their shared prefix through the tensor-memory kernel (prefix_flat_keys 0): the split-KV kernel
behind it starts while it runs, so what earlier kernels wrote - appended rows, queries, positions - has to be there.
Appended rows, captured and replayed steps, host-buffer steps and a layer's steps enqueued one behind the other."""
import numpy as np
import pytest
import torch

from test_gpu_layer_with_scores import Layer, capture
from test_gpu_shared_prefix import NAN, Step

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("heads,shared", [((8, 2), 260), ((16, 2), 5000), ((20, 1), 1300)], ids=str)
@pytest.mark.parametrize("starts", [[30, 2, 0], [(11 * b) % 300 for b in range(40)]], ids=["3", "40"])
def test_new_rows_are_appended(heads, shared, starts):
    s = Step(71, 1, starts, *heads, shared)
    want_k, want_v = s.k.clone(), s.v.clone()
    at = [s.starts[b] for b in range(s.B)]
    kn, vn = (torch.stack([c[b, :, at[b]] for b in range(s.B)])[None].contiguous() for c in (s.k, s.v))
    for b in range(s.B):
        s.k[b, :, at[b]:] = NAN
        s.v[b, :, at[b]:] = NAN
    op = s.op(k_new=kn, v_new=vn)
    op.set_option("prefix_flat_keys", 0)
    op.run_ragged(torch.tensor(s.starts, dtype=torch.int32, device=s.dev), 1, s.B)
    torch.cuda.synchronize()
    assert op.kernel_stats()["prefill_tcgen05"][0] == 1
    op.close()
    assert torch.equal(s.k.nan_to_num(3.0), want_k.nan_to_num(3.0)) and torch.equal(s.v.nan_to_num(3.0), want_v.nan_to_num(3.0))
    s.check()


@pytest.mark.parametrize("persistent", [-1, 0])
def test_captured_step_replays_with_new_inputs(persistent):
    s = Step(72, 1, [300, 20, 0] * 8, 16, 4, 2777)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        op = s.op(stream=stream.cuda_stream, async_=True)
        op.set_option("prefix_flat_keys", 0)
        op.set_option("tc_persistent", persistent)
        pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
        op.run_ragged(pos, 1, s.B)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            op.run_ragged(pos, 1, s.B)
        s.q.mul_(-0.5)
        s.pv.mul_(1.5)
        for _ in range(4):
            s.out.fill_(7.0)
            graph.replay()
        stream.synchronize()
    s.check()
    op.check()
    del graph
    op.close()


def test_host_buffer_steps_with_new_rows():
    s = Step(73, 1, [90, 17, 40, 3], 8, 2, 3150)
    kn, vn = (torch.zeros(1, s.B, s.Hkv, D, dtype=torch.bfloat16, device=s.dev) for _ in range(2))
    op = s.op(k_new=kn, v_new=vn)
    op.set_option("prefix_flat_keys", 0)
    qh, oh = s.q.cpu().pin_memory(), torch.zeros_like(s.out, device="cpu").pin_memory()
    ph, lh = torch.tensor(s.starts, dtype=torch.int32).pin_memory(), torch.zeros(s.lse.shape).pin_memory()
    knh, vnh = (torch.stack([c[b, :, s.starts[b]] for b in range(s.B)])[None].contiguous().cpu().pin_memory() for c in (s.k, s.v))
    s.q.zero_()
    for b in range(s.B):
        s.k[b, :, s.starts[b]] = NAN
        s.v[b, :, s.starts[b]] = NAN
    for _ in range(3):
        oh.zero_()
        op.run_host(qh, oh, 0, 1, s.B, positions_host=ph, lse_host=lh, k_new_host=knh, v_new_host=vnh)
    assert op.kernel_stats()["prefill_tcgen05"][0] == 3
    s.q.copy_(qh)
    s.out.copy_(oh)
    s.lse.copy_(lh)
    s.check()
    op.close()


@pytest.mark.parametrize("B,heads,hidden,shared", [(3, (8, 1), 384, 900), (24, (16, 4), 512, 3000)], ids=str)
@pytest.mark.parametrize("replayed", [False, True])
def test_steps_of_a_layer_one_behind_the_other(B, heads, hidden, shared, replayed):
    """Twelve decode steps with nothing waited for between them: projections write queries and new rows, attention
    appends and reads them, the positions are advanced on the device.  The last step is held against the reference
    over a cache that only the steps before it can have filled.  (The next input is tanh of the residual stream: the stream
    itself grows fourfold a step, and where scores reach 2e6 fp32 resolves 0.125, which no bar on the softmax can hold;
    the test below compares such steps bit by bit.)"""
    from ellm_b200 import _lib as L
    steps = 12
    layer = Layer(74, B, *heads, hidden, 100, 1)
    pk, pv = (torch.randn(2, heads[1], shared, D, generator=layer.gen) * 0.7).to(torch.bfloat16).to(layer.dev)
    layer.attn.set_shared_prefix(pk, pv)
    layer.attn.set_option("prefix_flat_keys", 0)
    starts = [(5 * b) % 17 for b in range(B)]
    rows = torch.randn(2, B, heads[1], 17, D, generator=layer.gen).to(torch.bfloat16).to(layer.dev)
    for b, p in enumerate(starts):                         # the history before the first step
        layer.cache[:, b, :, :p] = rows[:, b, :, :p]
    layer.load(1)
    lib = L.load()
    if replayed:
        layer.pos.fill_(90)
        layer.step(1)                                      # (before a capture every operator has run once)
        torch.cuda.synchronize()
        lib, graph, stream = capture(layer)
        layer.load(1)
    layer.pos.copy_(torch.tensor(starts, dtype=torch.int32))
    layer.cache[:, :, :, 90:] = NAN
    torch.cuda.synchronize()

    def step():
        if replayed:
            L.check(lib.ellm_step_graph_launch(graph, stream))
            return
        layer.step(1)
        L.check(lib.ellm_positions_set(layer.pos.data_ptr(), B, 1, 1, 0, layer.stream.cuda_stream))

    with torch.cuda.stream(layer.stream):
        for i in range(steps):
            step()
            layer.h.copy_(torch.tanh(layer.x))             # the next step's input
    torch.cuda.synchronize()
    starts = [p + steps for p in starts]
    assert layer.pos.tolist() == starts
    before, x_in = layer.cache.clone(), layer.load(1)
    for b, p in enumerate(starts):
        assert bool(torch.isfinite(before[:, b, :, :p].float()).all()) and bool(torch.isnan(before[:, b, :, p:].float()).all())
    step()

    def attend(b, pos):
        n = pos[-1] + 1
        return (torch.cat((pk, layer.cache[0, b, :, :n]), 1), torch.cat((pv, layer.cache[1, b, :, :n]), 1), np.zeros_like(pos),
                pos + 1 + shared, dict(shared=shared))
    layer.check(1, starts, before, x_in, attend)
    if replayed:
        L.check(lib.ellm_step_graph_destroy(graph))
    layer.close()


@pytest.mark.parametrize("replayed", [False, True])
def test_chained_steps_give_the_bits_of_steps_that_are_waited_for(replayed):
    """The same twelve steps, each waited for, end in the same residual stream, bit for bit."""
    from ellm_b200 import _lib as L
    lib, ends = L.load(), []
    for wait in (False, True):
        layer = Layer(75, 16, 16, 2, 512, 80, 1)
        pk, pv = (torch.randn(2, 2, 4000, D, generator=layer.gen) * 0.7).to(torch.bfloat16).to(layer.dev)
        layer.attn.set_shared_prefix(pk, pv)
        layer.attn.set_option("prefix_flat_keys", 0)
        layer.step(1)                                      # (before a capture every operator has run once)
        torch.cuda.synchronize()
        if replayed:
            lib, graph, stream = capture(layer)
        layer.load(1)
        layer.pos.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(layer.stream):
            for _ in range(12):
                if replayed:
                    L.check(lib.ellm_step_graph_launch(graph, stream))
                else:
                    layer.step(1)
                    L.check(lib.ellm_positions_set(layer.pos.data_ptr(), 16, 1, 1, 0, layer.stream.cuda_stream))
                layer.h.copy_(layer.x)
                if wait:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        ends.append((layer.x.clone(), layer.cache[:, :, :, :12].clone(), layer.lse.clone()))
        if replayed:
            L.check(lib.ellm_step_graph_destroy(graph))
        layer.close()
    assert all(torch.equal(a, b) for a, b in zip(*ends)) and bool(torch.isfinite(ends[0][0].float()).all())
