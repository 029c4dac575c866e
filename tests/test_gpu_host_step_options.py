"""Options of an attention handle that change between host-buffer decode steps: the captured step follows them."""
import pytest
import torch

from test_gpu_shared_prefix import Step as PrefixStep

pytestmark = pytest.mark.gpu


class HostStep:
    def __init__(self, seed, **kw):
        self.s = PrefixStep(seed, 1, [90, 17], 8, 2, 150)
        s = self.s
        self.op = s.op(**kw)
        self.q, self.out = s.q.cpu().pin_memory(), torch.zeros_like(s.out, device="cpu").pin_memory()
        self.pos, self.lse = torch.tensor(s.starts, dtype=torch.int32).pin_memory(), torch.zeros(s.lse.shape).pin_memory()

    def step(self):
        """One step; how often it launched the tensor-memory kernel."""
        before = self.op.kernel_stats()["prefill_tcgen05"][0]
        self.out.zero_()
        self.op.run_host(self.q, self.out, 0, 1, 2, positions_host=self.pos, lse_host=self.lse)
        self.s.out.copy_(self.out)
        self.s.lse.copy_(self.lse)
        self.s.check()
        return self.op.kernel_stats()["prefill_tcgen05"][0] - before


def test_the_kernel_chosen_for_the_prefix_follows_its_option():
    h = HostStep(51)
    h.op.set_option("prefix_flat_keys", 1 << 40)
    assert [h.step(), h.step()] == [0, 0]
    h.op.set_option("prefix_flat_keys", 0)
    assert [h.step(), h.step()] == [1, 1]
    h.op.set_option("prefix_flat_keys", 1 << 40)
    assert [h.step(), h.step()] == [0, 0]
    h.op.close()


def test_limits_and_hooks_set_after_the_first_step_take_effect():
    """A tile that never comes, asked for after the step was captured, is reported after the limit set then; taken back,
    the next step is right."""
    from ellm_b200 import EllmError
    from ellm_b200 import _lib as L
    h = HostStep(52)
    h.op.set_option("prefix_flat_keys", 0)
    assert h.step() == 1
    h.op.set_option("tc_wait_timeout_ns", 100_000_000)
    h.op.set_option("tc_debug_skip_kv_item", 1)
    with pytest.raises(EllmError) as e:
        h.step()
    assert e.value.status == L.ERR_DEVICE_TIMEOUT
    h.op.set_option("tc_debug_skip_kv_item", -1)
    assert [h.step(), h.step()] == [1, 1]
    h.op.close()
