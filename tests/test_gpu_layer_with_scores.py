"""The newer operators as a layer uses them, one stream, nothing waited for in between: 4-bit Q, K and V projections ->
attention (capped, biased and windowed scores; or a shared prefix) that appends the new rows -> 4-bit output projection
onto the residual stream.  A prompt chunk, then decode steps, eager and as one captured step replayed with positions
that the graph advances.  Every stage is held against the 64-bit form of its own inputs, so that the bars are the
stages' own and an error cannot hide behind another's."""
import ctypes as C

import numpy as np
import pytest
import torch

from operator_refs import assert_attention, assert_w4, attention_ref, w4_weights

pytestmark = pytest.mark.gpu
D = 128


class Layer:
    """hidden -> 4-bit projections and attention of B sequences; x [chunk, B, hidden] is the residual stream."""

    def __init__(self, seed, B, q_heads, kv_heads, hidden, max_seq, chunk, group=64):
        from ellm_b200 import Attention, MatMulAddW4, pack_int4
        g = torch.Generator().manual_seed(seed)
        dev = self.dev = torch.device("cuda:0")
        self.B, self.H, self.Hkv, self.hidden, self.max_seq, self.chunk, self.group = B, q_heads, kv_heads, hidden, max_seq, chunk, group
        self.gen = g
        self.stream = torch.cuda.Stream()

        def weights(n, k):
            q = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
            s = ((torch.rand(n, k // group, generator=g) + 0.5) * (0.4 / k ** 0.5)).to(torch.bfloat16)
            z = torch.randint(6, 10, (n, k // group), generator=g, dtype=torch.uint8)
            return tuple(t.to(dev) for t in (q, s, z))

        def buf(*shape, dtype=torch.bfloat16):
            return torch.zeros(*shape, dtype=dtype, device=dev)

        self.x = buf(chunk, B, hidden)
        self.h = buf(chunk, B, hidden)         # what the projections read (the stream itself is rewritten in place)
        self.q, self.att = buf(chunk, B, q_heads, D), buf(chunk, B, q_heads, D)
        self.kn, self.vn = buf(chunk, B, kv_heads, D), buf(chunk, B, kv_heads, D)
        self.cache = torch.full((2, B, kv_heads, max_seq, D), float("nan"), dtype=torch.bfloat16, device=dev)
        self.lse = buf(chunk, B, q_heads, dtype=torch.float32)
        self.w = {"q": weights(q_heads * D, hidden), "k": weights(kv_heads * D, hidden), "v": weights(kv_heads * D, hidden),
                  "o": weights(hidden, q_heads * D)}
        kw = dict(stream=self.stream.cuda_stream, async_=True)
        self.ops = []
        for name, dst in (("q", self.q), ("k", self.kn), ("v", self.vn)):
            q, s, z = self.w[name]
            self.ops.append(MatMulAddW4.new(self.h, pack_int4(q), s, None, dst, chunk * B, q.shape[0], hidden, group, zeros=z, max_batch=B, **kw))
        k, v = self.cache[0], self.cache[1]
        self.attn = Attention.new(self.q, k, v, self.att, B, q_heads, kv_heads, D, [k.stride(i) for i in range(4)], D ** -0.5,
                                  max_seq=max_seq, max_interval=chunk, lse=self.lse, k_new=self.kn, v_new=self.vn, **kw)
        q, s, z = self.w["o"]
        self.out = MatMulAddW4.new(self.att, pack_int4(q), s, self.x, self.x, chunk * B, hidden, q_heads * D, group, zeros=z, max_batch=B, **kw)
        self.pos = torch.zeros(B, dtype=torch.int32, device=dev)

    def step(self, rows):
        for op in self.ops:
            op.run(0, rows, self.B)
        self.attn.run_ragged(self.pos, rows, self.B)
        self.out.run(0, rows, self.B)

    def load(self, rows):
        new = torch.randn(rows, self.B, self.hidden, generator=self.gen).to(torch.bfloat16).to(self.dev)
        self.x[:rows], self.h[:rows] = new, new
        torch.cuda.synchronize()
        return new

    def check(self, rows, starts, before, x_in, attend):
        """`before`: the cache as it was; `attend(b, pos)` -> lo, hi, keyword arguments of the reference."""
        torch.cuda.synchronize()
        n = rows * self.B
        for op in self.ops + [self.out]:
            op.check()
        self.attn.check()
        for name, got in (("q", self.q), ("k", self.kn), ("v", self.vn)):
            q, s, z = self.w[name]
            assert_w4(got[:rows].reshape(n, -1), self.h[:rows].reshape(n, -1), w4_weights(q, s, z, self.group), None, rounded_weights=n > 32)
        want = before.clone()
        for b, p in enumerate(starts):
            want[0, b, :, p:p + rows] = self.kn[:rows, b].transpose(0, 1)
            want[1, b, :, p:p + rows] = self.vn[:rows, b].transpose(0, 1)
        assert torch.equal(self.cache.nan_to_num(9.0), want.nan_to_num(9.0))
        for b, p in enumerate(starts):
            pos = p + np.arange(rows)
            k, v, lo, hi, kw = attend(b, pos)
            ref, A, l = attention_ref(self.q[:rows, b], k, v, lo, hi, pos, D ** -0.5, **kw)
            assert_attention(self.att[:rows, b], ref, A, self.lse[:rows, b], l)
        q, s, z = self.w["o"]
        assert_w4(self.x[:rows].reshape(n, -1), self.att[:rows].reshape(n, -1), w4_weights(q, s, z, self.group), x_in.reshape(n, -1),
                  rounded_weights=n > 32)

    def close(self):
        for op in self.ops + [self.out, self.attn]:
            op.close()


def capture(layer):
    """One decode step with the positions advanced behind it, as a step graph."""
    from ellm_b200 import _lib as L
    lib, stream, graph = L.load(), C.c_void_p(layer.stream.cuda_stream), C.c_void_p()
    L.check(lib.ellm_step_graph_begin(0, stream))
    layer.step(1)
    L.check(lib.ellm_positions_set(layer.pos.data_ptr(), layer.B, 1, 1, 0, stream))
    L.check(lib.ellm_step_graph_end(0, stream, C.byref(graph)))
    return lib, graph, stream


@pytest.mark.parametrize("B,heads,hidden,prompt", [(1, (8, 2), 256, 70), (3, (8, 1), 384, 150), (20, (16, 4), 512, 33)], ids=str)
@pytest.mark.parametrize("kind", ["scores", "prefix"])
def test_prompt_then_decode_steps_eager_and_replayed(B, heads, hidden, prompt, kind):
    from ellm_b200 import _lib as L
    max_seq, window, cap, shared = 200, 48, 30.0, 300
    layer = Layer(1, B, *heads, hidden, max_seq, prompt)
    H, Hkv = heads
    if kind == "scores":
        slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=layer.dev)
        begin = torch.clamp(torch.arange(max_seq, dtype=torch.int32, device=layer.dev) - window + 1, min=0).repeat(B, 1).contiguous()
        layer.attn.set_scores(cap, slopes, begin)

        def attend(b, pos):
            n = pos[-1] + 1
            return layer.cache[0, b, :, :n], layer.cache[1, b, :, :n], np.maximum(pos - window + 1, 0), pos + 1, dict(cap=cap, slopes=slopes)
    else:
        pk, pv = (torch.randn(2, Hkv, shared, D, generator=layer.gen) * 0.7).to(torch.bfloat16).to(layer.dev)
        layer.attn.set_shared_prefix(pk, pv)

        def attend(b, pos):
            n = pos[-1] + 1
            return (torch.cat((pk, layer.cache[0, b, :, :n]), 1), torch.cat((pv, layer.cache[1, b, :, :n]), 1), np.zeros_like(pos),
                    pos + 1 + shared, dict(shared=shared))

    before, x_in = layer.cache.clone(), layer.load(prompt)
    layer.step(prompt)
    layer.check(prompt, [0] * B, before, x_in, attend)

    # sequences of different lengths from here on: decode continues at (and overwrites from) these positions
    starts = [prompt - 1 - (7 * b) % 30 for b in range(B)]
    layer.pos.copy_(torch.tensor(starts, dtype=torch.int32))
    before, x_in = layer.cache.clone(), layer.load(1)
    layer.step(1)
    layer.check(1, starts, before, x_in, attend)

    starts = [p + 1 for p in starts]
    layer.pos.copy_(torch.tensor(starts, dtype=torch.int32))
    torch.cuda.synchronize()
    lib, graph, stream = capture(layer)
    for _ in range(4):
        before, x_in = layer.cache.clone(), layer.load(1)
        L.check(lib.ellm_step_graph_launch(graph, stream))
        layer.check(1, starts, before, x_in, attend)
        starts = [p + 1 for p in starts]
        assert layer.pos.tolist() == starts
    L.check(lib.ellm_step_graph_destroy(graph))
    layer.close()
