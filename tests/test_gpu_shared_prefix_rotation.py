"""Rotated queries and keys behind a shared prefix.  The positions of a handle with a shared prefix count what follows it, and
the projection that rotates takes the same positions: it is given the table from row prefix_len on.  The suffix of a prompt
and a decode step computed that way give the bits of the same rows computed behind the whole prompt in one cache, and
attention over prefix and own rows is attention over that cache."""
import numpy as np
import pytest
import torch

from operator_refs import assert_attention, attention_ref

pytestmark = pytest.mark.gpu
D, HIDDEN = 128, 256


class Model:
    """Projection (heads normalised and rotated, K and V written into the cache) and attention of one layer."""

    def __init__(self, w, rope, batch, heads, kv_heads, max_seq, interval):
        from ellm_b200 import Attention, MatMul3
        dev = w.device
        self.x = torch.zeros(interval, batch, HIDDEN, dtype=torch.bfloat16, device=dev)
        self.q = torch.zeros(interval, batch, heads, D, dtype=torch.bfloat16, device=dev)
        self.out, self.lse = torch.zeros_like(self.q), torch.zeros(interval, batch, heads, device=dev)
        self.k, self.v = torch.full((2, batch, kv_heads, max_seq, D), float("nan"), dtype=torch.bfloat16, device=dev)
        strides = [self.k.stride(i) for i in range(4)]
        wq, wk, wv = w[:heads * D], w[heads * D:(heads + kv_heads) * D], w[(heads + kv_heads) * D:]
        self.proj = MatMul3.new(self.x, wq, self.q, wk, self.k, wv, self.v, rope, D, interval * batch, HIDDEN, heads * D, kv_heads * D,
                                kv_strides=strides, max_batch=batch, max_seq=max_seq, rope_rows=rope.shape[0])
        self.attn = Attention.new(self.q, self.k, self.v, self.out, batch, heads, kv_heads, D, strides, D ** -0.5, max_seq=max_seq,
                                  max_interval=interval, lse=self.lse)
        self.batch = batch

    def step(self, x, position, prefix=None):
        self.x[:x.shape[0]] = x
        torch.cuda.synchronize()
        self.proj.run(position, x.shape[0], self.batch)
        if prefix is not None:
            self.attn.set_shared_prefix(*prefix)
        self.attn.run(position, x.shape[0], self.batch)
        torch.cuda.synchronize()
        return self.q[:x.shape[0]].clone(), self.out[:x.shape[0]].clone(), self.lse[:x.shape[0]].clone()


@pytest.mark.parametrize("prefix", [1, 150, 515])
@pytest.mark.parametrize("B,heads", [(1, (4, 4)), (3, (8, 2))], ids=str)
def test_suffix_and_decode_step_behind_a_prefix(prefix, B, heads):
    import ellm_b200
    H, Hkv = heads
    rows, total = 40, prefix + 48
    g = torch.Generator().manual_seed(91)
    dev = torch.device("cuda:0")
    w = (torch.randn((H + 2 * Hkv) * D, HIDDEN, generator=g) * 0.06).to(torch.bfloat16).to(dev)
    rope = torch.from_numpy(ellm_b200.precompute_freqs_cis(D, total, 1e4)).to(dev)
    shared_x = torch.randn(prefix, 1, HIDDEN, generator=g).to(torch.bfloat16).to(dev)
    suffix_x, step_x = (torch.randn(n, B, HIDDEN, generator=g).to(torch.bfloat16).to(dev) for n in (rows, 1))

    whole = Model(w, rope, B, H, Hkv, total, max(prefix, rows))      # every sequence with the prompt in its own cache
    whole.step(shared_x.expand(-1, B, -1), 0)
    behind = Model(w, rope[prefix:], B, H, Hkv, 48, rows)
    pk, pv = whole.k[0, :, :prefix].clone(), whole.v[0, :, :prefix].clone()
    for x, at in ((suffix_x, 0), (step_x, rows)):
        want_q, _, _ = whole.step(x, prefix + at)
        q, out, lse = behind.step(x, at, (pk, pv))
        n = x.shape[0]
        assert torch.equal(q, want_q)
        for own, full in ((behind.k, whole.k), (behind.v, whole.v)):
            assert torch.equal(own[:, :, :at + n], full[:, :, prefix:prefix + at + n])
        pos = prefix + at + np.arange(n)
        for b in range(B):
            end = prefix + at + n
            ref, A, l = attention_ref(q[:, b], whole.k[b, :, :end], whole.v[b, :, :end], np.zeros_like(pos), pos + 1, pos, D ** -0.5)
            assert_attention(out[:, b], ref, A, lse[:, b], l)
    for m in (whole, behind):
        m.proj.close()
        m.attn.close()
