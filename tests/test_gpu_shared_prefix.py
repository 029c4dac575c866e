"""Attention of a batch whose sequences share a prefix kept once (Attention.set_shared_prefix), against a 64-bit
reference over the prefix keys followed by each sequence's own."""
import numpy as np
import pytest
import torch

from operator_refs import assert_attention, attention_ref

pytestmark = pytest.mark.gpu
D = 128
NAN = float("nan")


class Step:
    def __init__(self, seed, rows, starts, q_heads, kv_heads, shared, max_seq=None, max_batch=None, seq_major=False,
                 spare=5, sharp=2.0):
        g = torch.Generator().manual_seed(seed)
        dev = self.dev = torch.device("cuda:0")
        self.rows, self.starts, self.H, self.Hkv, self.P = rows, list(starts), q_heads, kv_heads, shared
        self.B, self.mb = len(starts), max_batch or len(starts)
        self.max_seq = max_seq or max(starts) + rows + 3
        self.q = (torch.randn(rows, self.mb, q_heads, D, generator=g) * sharp).to(torch.bfloat16).to(dev)
        own = torch.randn(2, self.mb, kv_heads, self.max_seq, D, generator=g).to(torch.bfloat16)
        for b in range(self.mb):
            own[:, b, :, (max(0, self.starts[b] + rows) if b < self.B else 0):] = NAN
        pre = torch.randn(2, kv_heads, shared + spare, D, generator=g).to(torch.bfloat16)
        pre[:, :, shared:] = NAN                      # rows past the prefix are never read
        own, pre = own.to(dev), pre.to(dev)
        if seq_major:
            own = own.permute(0, 3, 1, 2, 4).contiguous().permute(0, 2, 3, 1, 4)
            pre = pre.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        self.k, self.v, self.pk, self.pv = own[0], own[1], pre[0], pre[1]
        self.strides = [self.k.stride(i) for i in range(4)]
        self.out = torch.full((rows, self.mb, q_heads, D), 7.0, dtype=torch.bfloat16, device=dev)
        self.lse = torch.full((rows, self.mb, q_heads), 7.0, device=dev)

    def op(self, prefill_kernel=0, **kw):
        from ellm_b200 import Attention
        op = Attention.new(self.q, self.k, self.v, self.out, self.mb, self.H, self.Hkv, D, self.strides, D ** -0.5,
                           max_seq=self.max_seq, max_interval=self.rows, lse=self.lse, prefill_kernel=prefill_kernel, **kw)
        op.set_shared_prefix(self.pk, self.pv, self.P)
        return op

    def run(self, prefill_kernel=0, ragged=None):
        op = self.op(prefill_kernel)
        if (len(set(self.starts)) > 1) if ragged is None else ragged:
            op.run_ragged(torch.tensor(self.starts, dtype=torch.int32, device=self.dev), self.rows, self.B)
        else:
            op.run(self.starts[0], self.rows, self.B)
        torch.cuda.synchronize()
        op.close()
        return self

    def check(self):
        for b in range(self.B):
            pos = self.starts[b] + np.arange(self.rows)
            n = max(0, self.starts[b] + self.rows)
            k = torch.cat((self.pk[:, :self.P], self.k[b, :, :n]), 1)
            v = torch.cat((self.pv[:, :self.P], self.v[b, :, :n]), 1)
            ref, A, l = attention_ref(self.q[:, b], k, v, np.zeros_like(pos), pos + 1 + self.P, pos, D ** -0.5, shared=self.P)
            assert_attention(self.out[:, b], ref, A, self.lse[:, b], l)
        assert bool((self.out[:, self.B:] == 7.0).all()) and bool((self.lse[:, self.B:] == 7.0).all())
        return self


@pytest.mark.parametrize("shared", [1, 127, 128, 129, 1000, 2049])
@pytest.mark.parametrize("starts", [[0], [5, 64, 200], list(range(0, 40, 2))], ids=["1", "3", "20"])
def test_decode(shared, starts):
    Step(1, 1, starts, 16, 2, shared).run(ragged=True).check()


@pytest.mark.parametrize("heads", [(4, 4), (5, 1), (14, 2), (24, 2), (64, 1), (160, 1)], ids=str)
def test_decode_groups(heads):
    Step(2, 1, [3, 77, 12, 0, 130], *heads, shared=700, max_batch=7).run().check()


@pytest.mark.parametrize("batch", [1, 15, 16, 17, 31, 32, 33, 64, 130])
def test_decode_batches(batch):
    Step(3, 1, [(7 * b) % 50 for b in range(batch)], 8, 1, shared=900).run(ragged=True).check()


def test_decode_long_prefix_uniform_positions_and_prefix_alone():
    Step(4, 1, [9, 9, 9, 9], 32, 4, shared=20011).run().check()
    Step(5, 1, [-1, 4, -1], 16, 4, shared=333).run().check()


def test_decode_leaping_scores_in_every_part():
    s = Step(6, 1, [40, 50, 60, 70], 8, 1, shared=5000, sharp=1.0)
    for key, f in ((100, 10.0), (2500, 20.0), (4999, 40.0)):
        s.pk[:, key] = (s.q[0, 1, 0] * f).to(torch.bfloat16)
    s.k[2, :, 55] = (s.q[0, 2, 3] * 50).to(torch.bfloat16)
    s.run().check()


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("shared", [1, 64, 128, 500, 1025])
@pytest.mark.parametrize("rows,starts", [(2, [0, 0]), (60, [0, 100, 31]), (200, [128])], ids=str)
def test_chunk(kernel, shared, rows, starts):
    Step(7, rows, starts, 16, 2, shared, max_batch=len(starts) + 1).run(kernel).check()


@pytest.mark.parametrize("kernel", [0, 2])
@pytest.mark.parametrize("heads", [(3, 3), (5, 1), (14, 2), (64, 1), (100, 1)], ids=str)
def test_chunk_groups(kernel, heads):
    Step(8, 33, [0, 17], *heads, shared=200).run(kernel).check()


@pytest.mark.parametrize("rows", [1, 40])
def test_seq_major_strides(rows):
    Step(9, rows, [0, 20, 90], 8, 2, 300, seq_major=True).run().check()


@pytest.mark.parametrize("rows", [1, 50])
def test_new_rows_are_appended_to_the_own_cache(rows):
    s = Step(10, rows, [30, 2, 0], 8, 2, 260)
    want_k, want_v = s.k.clone(), s.v.clone()
    kn = torch.stack([torch.stack([s.k[b, :, s.starts[b] + r] for b in range(3)]) for r in range(rows)]).contiguous()
    vn = torch.stack([torch.stack([s.v[b, :, s.starts[b] + r] for b in range(3)]) for r in range(rows)]).contiguous()
    for b in range(3):
        s.k[b, :, s.starts[b]:] = NAN
        s.v[b, :, s.starts[b]:] = NAN
    op = s.op(k_new=kn, v_new=vn)
    op.run_ragged(torch.tensor(s.starts, dtype=torch.int32, device=s.dev), rows, 3)
    torch.cuda.synchronize()
    op.close()
    assert torch.equal(s.k.nan_to_num(3.0), want_k.nan_to_num(3.0)) and torch.equal(s.v.nan_to_num(3.0), want_v.nan_to_num(3.0))
    s.check()


def test_the_prefix_may_be_a_slot_of_the_same_cache_and_be_swapped_and_removed():
    from ellm_b200 import Attention
    s = Step(11, 1, [10, 20], 8, 2, 100)
    op = s.op()
    pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
    op.run_ragged(pos, 1, 2)
    torch.cuda.synchronize()
    s.check()
    s.pk, s.pv, s.P = s.k[0, :, :9].clone(), s.v[0, :, :9].clone(), 9
    op.set_shared_prefix(s.k[0], s.v[0], 9)
    op.run_ragged(pos, 1, 2)
    torch.cuda.synchronize()
    s.check()
    op.set_shared_prefix(None, None)
    op.run_ragged(pos, 1, 2)
    torch.cuda.synchronize()
    s.P = 0
    s.check()
    op.close()


@pytest.mark.parametrize("rows", [1, 70])
def test_captured_step_replays_with_new_inputs(rows):
    s = Step(12, rows, [300, 20, 0], 16, 4, 777)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        op = s.op(stream=stream.cuda_stream, async_=True)
        pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
        op.run_ragged(pos, rows, 3)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            op.run_ragged(pos, rows, 3)
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


def test_host_buffer_step():
    s = Step(13, 1, [90, 17], 8, 2, 150)
    op = s.op()
    qh, oh = s.q.cpu().pin_memory(), torch.zeros_like(s.out, device="cpu").pin_memory()
    ph, lh = torch.tensor(s.starts, dtype=torch.int32).pin_memory(), torch.zeros(s.lse.shape).pin_memory()
    s.q.zero_()
    for _ in range(3):
        oh.zero_()
        op.run_host(qh, oh, 0, 1, 2, positions_host=ph, lse_host=lh)
    s.q.copy_(qh)
    s.out.copy_(oh)
    s.lse.copy_(lh)
    s.check()
    op.close()


def test_refusals():
    from ellm_b200 import EllmError
    s = Step(14, 4, [0], 8, 2, 20)
    op = s.op()
    part, lse = torch.zeros(4, 1, 8, D, device=s.dev), torch.zeros(4, 1, 8, device=s.dev)
    with pytest.raises(EllmError):
        op.run_window(0, 4, 1, 0, 4, part, lse)
    with pytest.raises(EllmError):
        op.set_scores(softcap=3.0)
    op.set_scores()                                   # nothing to take back: the prefix stays
    with pytest.raises(ValueError):
        op.set_shared_prefix(s.pk.float(), s.pv.float(), 4)
    with pytest.raises(ValueError):
        op.set_shared_prefix(s.pk[:1], s.pv[:1], 4)
    with pytest.raises(ValueError):
        op.set_shared_prefix(s.pk, s.pv, 1000)
    with pytest.raises(ValueError):
        op.set_shared_prefix(s.pk.data_ptr(), s.pv.data_ptr())
    with pytest.raises(EllmError):
        op.set_shared_prefix(s.pk.data_ptr(), s.pv.data_ptr() + 2, 4, (1024, 128))
    with pytest.raises(EllmError):
        op.set_shared_prefix(s.pk.data_ptr(), s.pv.data_ptr(), 4, (1024, 100))
    with pytest.raises(EllmError):
        op.set_shared_prefix(s.pk.data_ptr(), None, 4, (1024, 128))
    op.run(0, 4, 1)
    torch.cuda.synchronize()
    s.check()
    op.close()
