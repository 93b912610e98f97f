"""Block copies between tensors that share memory: the same tensor with other
blocks, or refused."""
import pytest
import torch

from rlx_models_b200 import ops


def test_a_shared_tensor_behind_one_of_its_own():
    """The first pair of tensors is apart, the second is one tensor: its destination is also a source."""
    a, b, k = (torch.zeros(2, 5, 3) for _ in range(3))
    with pytest.raises(ValueError, match="also a source"):
        ops.kv_copy_blocks([a, k], [b, k], [0, 1], [1, 2])


@pytest.mark.gpu
def test_overlapping_views_are_refused(cuda):
    k = torch.arange(240., device=cuda).view(4, 5, 12)
    before = k.clone()
    line = k.view(1, 20, 12)
    other = torch.zeros_like(k)
    for src, dst in (([k[:3]], [k[1:]]),                       # one layer further on
                     ([line[:, :10]], [line[:, 5:15]]),        # blocks further on
                     ([k, other], [other, k]),                 # crosswise
                     ([k, k], [other, other]),                 # two parts into one
                     ([k[:, :, :6].contiguous()] * 2, [other.view(-1)[:120].view(4, 5, 6),
                                                       other.view(-1)[60:180].view(4, 5, 6)])):
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.kv_copy_blocks(src, dst, [0], [1])
    assert torch.equal(k, before) and not bool(other.any())
    ops.kv_copy_blocks([k, other], [k, other], [0, 3], [1, 4])
    ops.kv_copy_blocks([line[:, :10]], [line[:, 10:]], [2], [3])
    want = before.clone()
    want[:, [1, 4]] = want[:, [0, 3]]
    want.view(1, 20, 12)[:, 13] = want.view(1, 20, 12)[:, 2]
    ops.check_errors(cuda)
    assert torch.equal(k, want)
