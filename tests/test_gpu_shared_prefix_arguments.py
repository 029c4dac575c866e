"""Arguments of Attention.set_shared_prefix that the Python mirror refuses before they reach the library."""
import pytest
import torch

from test_gpu_shared_prefix import Step

D = 128


def test_keys_and_values_come_in_one_form():
    from ellm_b200 import Attention
    from ellm_b200 import _lib as L
    op = object.__new__(Attention)
    op._h, op.desc = None, L.AttnDesc()
    op.desc.q_heads, op.desc.kv_heads, op.desc.head_size, op.desc.max_batch, op.desc.max_seq = 8, 2, D, 3, 40
    kv = torch.zeros(2, 9, D, dtype=torch.bfloat16)
    for k, v in ((kv, None), (kv, 0x1000), (0x1000, kv)):
        with pytest.raises(ValueError, match="both be tensors or both raw pointers"):
            op.set_shared_prefix(k, v, 9, (9 * D, D))


@pytest.mark.gpu
def test_strides_of_tensors_are_their_own():
    s = Step(111, 1, [5, 3], 8, 2, 40)
    op = s.op()
    own = (s.pk.stride(0), s.pk.stride(1))
    for strides in ((own[0] * 2, own[1]), (own[0], own[1] * 2), (1 << 30, D)):
        with pytest.raises(ValueError, match="strides go with raw pointers"):
            op.set_shared_prefix(s.pk, s.pv, 40, strides)
    op.set_shared_prefix(s.pk, s.pv, 40, own)
    op.run_ragged(torch.tensor(s.starts, dtype=torch.int32, device=s.dev), 1, 2)
    torch.cuda.synchronize()
    s.check()
    op.close()
