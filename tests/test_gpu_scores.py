"""Attention with capped and biased scores and one key interval per row (Attention.set_scores) against a 64-bit
reference: decode steps, chunks on both chunk kernels, masks that leave rows empty, what masked keys hold."""
import numpy as np
import pytest
import torch

from operator_refs import assert_attention, attention_ref

pytestmark = pytest.mark.gpu
D = 128
NAN = float("nan")


class Step:
    """One operator over a cache whose rows past every sequence's end are NaN."""

    def __init__(self, seed, rows, starts, q_heads, kv_heads, max_seq, max_batch=None, seq_major=False, sharp=2.0):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.starts, self.H, self.Hkv, self.max_seq = rows, list(starts), q_heads, kv_heads, max_seq
        self.B, self.mb = len(starts), max_batch or len(starts)
        dev = self.dev = torch.device("cuda:0")
        self.q = (torch.randn(rows, self.mb, q_heads, D, generator=g) * sharp).to(torch.bfloat16).to(dev)
        kv = torch.randn(2, self.mb, kv_heads, max_seq, D, generator=g).to(torch.bfloat16)
        for b in range(self.mb):
            kv[:, b, :, (self.starts[b] + rows if b < self.B else 0):] = NAN
        kv = kv.to(dev)
        if seq_major:      # [position, sequence, head]: the stride order of a max-shape activation buffer
            kv = kv.permute(0, 3, 1, 2, 4).contiguous().permute(0, 2, 3, 1, 4)
        self.k, self.v = kv[0], kv[1]
        self.strides = [self.k.stride(i) for i in range(4)]
        self.out = torch.full((rows, self.mb, q_heads, D), 7.0, dtype=torch.bfloat16, device=dev)
        self.lse = torch.full((rows, self.mb, q_heads), 7.0, device=dev)
        self.cap, self.slopes, self.begin, self.prefix = 0.0, None, None, None

    def scores(self, cap=0.0, bias=False, begin=None, prefix=None):
        self.cap = cap
        if bias:
            self.slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / self.H) for h in range(self.H)], device=self.dev)
        if begin is not None:
            self.begin = torch.as_tensor(np.asarray(begin, dtype=np.int32)).to(self.dev)
        if prefix is not None:
            self.prefix = torch.as_tensor(np.asarray(prefix, dtype=np.int32)).to(self.dev)
        return self

    def op(self, prefill_kernel=0, **kw):
        from ellm_b200 import Attention
        op = Attention.new(self.q, self.k, self.v, self.out, self.mb, self.H, self.Hkv, D, self.strides, D ** -0.5,
                           max_seq=self.max_seq, max_interval=self.rows, lse=self.lse, prefill_kernel=prefill_kernel, **kw)
        op.set_scores(self.cap, self.slopes, self.begin, self.prefix)
        return op

    def run(self, prefill_kernel=0, ragged=None):
        op = self.op(prefill_kernel)
        ragged = len(set(self.starts)) > 1 if ragged is None else ragged
        if ragged:
            op.run_ragged(torch.tensor(self.starts, dtype=torch.int32, device=self.dev), self.rows, self.B)
        else:
            op.run(self.starts[0], self.rows, self.B)
        torch.cuda.synchronize()
        self.stats = op.kernel_stats()
        op.close()
        return self

    def intervals(self, b):
        pos = self.starts[b] + np.arange(self.rows)
        lo = np.maximum(self.begin[b].cpu().numpy()[pos], 0) if self.begin is not None else np.zeros_like(pos)
        hi = pos + 1
        if self.prefix is not None:
            hi = np.maximum(hi, int(self.prefix[b]))
        return pos, lo, np.minimum(hi, self.starts[b] + self.rows)

    def check(self, lse=True):
        for b in range(self.B):
            pos, lo, hi = self.intervals(b)
            ref, A, l = attention_ref(self.q[:, b], self.k[b], self.v[b], lo, hi, pos, D ** -0.5, self.cap, self.slopes)
            assert_attention(self.out[:, b], ref, A, self.lse[:, b] if lse else None, l)
        assert bool((self.out[:, self.B:] == 7.0).all()) and bool((self.lse[:, self.B:] == 7.0).all())
        return self


def windows(batch, max_seq, w):
    return np.repeat(np.maximum(np.arange(max_seq) - w + 1, 0)[None], batch, 0)


def documents(seed, batch, max_seq, mean):
    rng = np.random.default_rng(seed)
    out = np.zeros((batch, max_seq), dtype=np.int32)
    for b in range(batch):
        at = 0
        while at < max_seq:
            n = int(rng.integers(1, 2 * mean + 1))
            out[b, at:at + n] = at
            at += n
    return out


# -------------------------------------------------------------------------------------------------- decode
@pytest.mark.parametrize("heads", [(8, 8), (8, 1), (10, 2), (14, 2), (32, 2), (40, 2)], ids=str)
@pytest.mark.parametrize("cap,bias", [(50.0, False), (0.0, True), (3.0, True)])
def test_decode_ragged(heads, cap, bias):
    Step(11, 1, [0, 62, 63, 64, 200, 1037], *heads, max_seq=1100, max_batch=8).scores(cap, bias).run().check()


@pytest.mark.parametrize("window", [1, 16, 63, 64, 65, 500])
def test_decode_window(window):
    s = Step(12, 1, [0, 5, 64, 700, 1500], 16, 4, max_seq=1600)
    s.scores(30.0, True, begin=windows(5, 1600, window)).run().check()


def test_decode_uniform_single_and_empty_rows():
    Step(13, 1, [0], 32, 4, max_seq=8).scores(50.0).run().check()
    s = Step(14, 1, [10, 300, 0], 16, 4, max_seq=320)
    begin = np.zeros((3, 320), dtype=np.int32)
    begin[0, 10] = 11          # sees nothing
    begin[1, 300] = 300        # itself alone
    begin[2, 0] = -5           # counts as 0
    s.scores(0.0, False, begin=begin).run().check()
    assert bool((s.out[0, 0] == 0).all()) and bool(torch.isneginf(s.lse[0, 0]).all())


def test_decode_large_batch_and_many_pieces():
    rng = np.random.default_rng(5)
    Step(15, 1, rng.integers(0, 190, 150), 8, 2, max_seq=200).scores(20.0, True).run().check()
    Step(16, 1, [16000], 8, 1, max_seq=16001).scores(50.0, True, begin=windows(1, 16001, 12345)).run().check()


# --------------------------------------------------------------------------------------------------- chunks
KERNELS = [1, 2]     # tcgen05, warp MMA


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("rows,starts", [(2, [0]), (17, [0, 0]), (129, [77]), (300, [0, 130, 511])], ids=str)
@pytest.mark.parametrize("cap,bias", [(50.0, False), (0.0, True), (4.0, True), (0.0, False)])
def test_chunk_causal(kernel, rows, starts, cap, bias):
    begin = None if cap or bias else np.zeros((len(starts), 900), dtype=np.int32)
    Step(21, rows, starts, 16, 2, max_seq=900).scores(cap, bias, begin).run(kernel).check()


@pytest.mark.parametrize("kernel", [0, 2])
@pytest.mark.parametrize("heads", [(3, 3), (5, 1), (14, 2), (24, 2), (64, 1), (100, 1)], ids=str)
def test_chunk_groups(kernel, heads):
    Step(22, 70, [0, 40], *heads, max_seq=128).scores(20.0, True, begin=documents(1, 2, 128, 30)).run(kernel).check()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("mean", [1, 20, 150, 600])
def test_chunk_documents_and_padding(kernel, mean):
    begin = documents(mean, 2, 700, mean)
    begin[0, 650:] = np.arange(651, 701)      # padded rows at the end see nothing
    begin[1, :9] = np.arange(1, 10)           # and at the start
    begin[1, 9:][begin[1, 9:] < 9] = 9
    s = Step(23, 700, [0, 0], 8, 2, max_seq=700).scores(0.0, True, begin=begin).run(kernel).check()
    assert bool((s.out[650:, 0] == 0).all()) and bool((s.out[:9, 1] == 0).all())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("window", [1, 100, 128, 129, 1000])
def test_chunk_window_later_piece(kernel, window):
    Step(24, 260, [600, 333, 0], 8, 1, max_seq=900).scores(50.0, False, begin=windows(3, 900, window)).run(kernel).check()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("prefix", [[1, 0, 300], [128, 129, 7], [500, 255, 256]], ids=str)
def test_chunk_prefix_mask(kernel, prefix):
    Step(25, 300, [0, 0, 0], 16, 4, max_seq=305).scores(50.0, True, prefix=prefix).run(kernel).check()


@pytest.mark.parametrize("kernel", KERNELS)
def test_chunk_prefix_mask_over_documents_and_ragged_starts(kernel):
    s = Step(26, 200, [0, 150], 8, 2, max_seq=400)
    s.scores(10.0, True, begin=documents(9, 2, 400, 90), prefix=[120, 333]).run(kernel).check()


@pytest.mark.parametrize("kernel", KERNELS)
def test_chunk_strides_and_idle_sequence_slots(kernel):
    Step(27, 150, [0, 20], 8, 2, max_seq=190, max_batch=4, seq_major=True).scores(50.0, True).run(kernel).check()


@pytest.mark.parametrize("kernel", KERNELS)
def test_chunk_many_tiles_with_leaping_scores(kernel):
    """A few keys whose scores tower over the rest, behind the first tiles: the rescaling paths."""
    s = Step(28, 384, [1200], 8, 1, max_seq=1600, sharp=1.0)
    for key, f in ((200, 12.0), (333, 25.0), (1000, 40.0), (1100, 60.0)):
        s.k[0, :, key] = (s.q[5, 0, 0] * f).to(torch.bfloat16)
    s.scores(60.0).run(kernel).check()
    s.scores(0.0, True).run(kernel).check()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")], ids=str)
def test_masked_keys_may_hold_anything(kernel, value):
    """Keys of one document (and of padding) are NaN or infinite; the other documents' rows never see them."""
    s = Step(29, 400, [0], 8, 2, max_seq=400)
    begin = np.zeros((1, 400), dtype=np.int32)
    begin[0, 90:] = 90
    begin[0, 213:] = 213
    s.scores(20.0, True, begin=begin)
    s.k[0, :, 100:213] = value
    s.v[0, :, 95:200] = value
    s.run(kernel)
    pos, lo, hi = s.intervals(0)
    ref, A, l = attention_ref(s.q[:, 0], s.k[0], torch.nan_to_num(s.v[0], 0.0, 0.0, 0.0), lo, hi, pos, D ** -0.5, 20.0, s.slopes)
    for r in (slice(0, 90), slice(213, 400)):
        assert_attention(s.out[r, 0], ref[r], A[r], s.lse[r, 0], l[r])


def test_chunk_kernels_agree_with_plain_attention_when_nothing_is_set():
    from ellm_b200 import Attention
    s = Step(30, 333, [0], 16, 2, max_seq=333)
    op = s.op()
    op.run(0, 333, 1)
    torch.cuda.synchronize()
    plain = s.out.clone()
    op.set_scores(softcap=1e6)
    op.run(0, 333, 1)
    torch.cuda.synchronize()
    assert (s.out.float() - plain.float()).abs().max().item() <= 2e-2
    op.set_scores()                           # back to plain attention: the same bits as before
    s.out.fill_(7.0)
    op.run(0, 333, 1)
    torch.cuda.synchronize()
    assert torch.equal(s.out, plain)
    op.close()


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("masked", [False, True])
def test_new_rows_are_appended(rows, masked):
    from ellm_b200 import Attention
    s = Step(31, rows, [40, 0], 8, 2, max_seq=300)
    want_k, want_v = s.k.clone(), s.v.clone()
    kn = torch.stack([torch.stack([s.k[b, :, s.starts[b] + r] for b in range(2)]) for r in range(rows)]).contiguous()
    vn = torch.stack([torch.stack([s.v[b, :, s.starts[b] + r] for b in range(2)]) for r in range(rows)]).contiguous()
    for b in range(2):
        s.k[b, :, s.starts[b]:] = NAN
        s.v[b, :, s.starts[b]:] = NAN
    begin = None
    if masked:
        begin = np.zeros((2, 300), dtype=np.int32)
        begin[1, :] = np.arange(1, 301)        # a sequence whose rows see nothing still gets its rows stored
    s.scores(30.0, False, begin)
    op = s.op(k_new=kn, v_new=vn)
    op.run_ragged(torch.tensor(s.starts, dtype=torch.int32, device=s.dev), rows, 2)
    torch.cuda.synchronize()
    op.close()
    assert torch.equal(s.k.nan_to_num(3.0), want_k.nan_to_num(3.0)) and torch.equal(s.v.nan_to_num(3.0), want_v.nan_to_num(3.0))
    s.check()


def test_host_buffer_steps_follow_a_change_of_the_scores():
    s = Step(32, 1, [90, 17], 8, 2, max_seq=128)
    op = s.scores(5.0).op()
    qh, oh = s.q.cpu().pin_memory(), torch.zeros_like(s.out, device="cpu").pin_memory()
    ph = torch.tensor(s.starts, dtype=torch.int32).pin_memory()
    lh = torch.zeros(s.lse.shape).pin_memory()
    for cap, bias in ((5.0, False), (5.0, True), (0.0, False)):
        s.slopes = None
        s.scores(cap, bias)
        op.set_scores(s.cap, s.slopes)
        for _ in range(2):
            oh.zero_()
            op.run_host(qh, oh, 0, 1, 2, positions_host=ph, lse_host=lh)
        s.out.copy_(oh)
        s.lse.copy_(lh)
        s.check()
    op.close()


@pytest.mark.parametrize("rows", [1, 160])
def test_captured_step_replays_with_new_inputs(rows):
    s = Step(33, rows, [300, 20], 16, 4, max_seq=500).scores(30.0, True, begin=documents(2, 2, 500, 70))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        op = s.op(stream=stream.cuda_stream, async_=True)
        pos = torch.tensor(s.starts, dtype=torch.int32, device=s.dev)
        op.run_ragged(pos, rows, 2)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            op.run_ragged(pos, rows, 2)
        s.q.mul_(-0.5)
        s.begin.copy_(torch.from_numpy(documents(3, 2, 500, 20)))
        for _ in range(3):
            s.out.fill_(7.0)
            graph.replay()
        stream.synchronize()
    s.check()
    op.check()
    del graph
    op.close()


def test_refusals():
    from ellm_b200 import EllmError
    s = Step(34, 4, [0], 8, 2, max_seq=64)
    op = s.op()
    part = torch.zeros(4, 1, 8, D, device=s.dev)
    lse = torch.zeros(4, 1, 8, device=s.dev)
    ok = torch.zeros(8, device=s.dev)
    with pytest.raises(EllmError):
        op.set_scores(softcap=-1.0)
    with pytest.raises(EllmError):
        op.set_scores(softcap=float("nan"))
    with pytest.raises(EllmError):
        op.set_scores(softcap=float("inf"))
    with pytest.raises(ValueError):
        op.set_scores(slopes=ok[:4])
    with pytest.raises(ValueError):
        op.set_scores(slopes=ok.double())
    with pytest.raises(ValueError):
        op.set_scores(slopes=ok.cpu())
    with pytest.raises(ValueError):
        op.set_scores(row_begin=torch.zeros(1, 63, dtype=torch.int32, device=s.dev))
    with pytest.raises(ValueError):
        op.set_scores(row_begin=torch.zeros(1, 64, dtype=torch.int64, device=s.dev))
    with pytest.raises(ValueError):
        op.set_scores(prefix_lens=torch.zeros(2, dtype=torch.int32, device=s.dev))
    op.run(0, 4, 1)                            # a refused call leaves the operator as it was
    op.set_scores(softcap=2.0)
    with pytest.raises(EllmError):
        op.run_window(0, 4, 1, 0, 4, part, lse)
    with pytest.raises(EllmError):
        op.set_shared_prefix(s.k[0], s.v[0], 10)
    op.set_scores()
    op.run_window(0, 4, 1, 0, 4, part, lse)
    op.close()
