"""Host-side checks of the int8 KV cache and draft verification: the 64-bit
oracles against hand-worked values, and arguments refused before any launch."""
import pytest
import torch

from rlx_models_b200 import ops
from rlx_models_b200.ops import reference as ref


def test_scale_is_the_smallest_power_of_two():
    assert ref.pow2_scale(0.0) == 2.0 ** -100
    assert ref.pow2_scale(127.0) == 1.0 and ref.pow2_scale(127.5) == 2.0
    assert ref.pow2_scale(1.0) == 2.0 ** -6 and ref.pow2_scale(1.9921875) == 2.0 ** -5


def test_store_oracle_by_hand():
    codes, scale = torch.full((2, 1, 16, 64), 50, dtype=torch.int8), torch.full((2, 1), 0.25)
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    x[0, 0, 0], x[1, 0, 0] = 10.0, -100.0  # 10 fits the old scale, 100 needs 1.0: codes 50 -> round(12.5) = 12
    ref.store_int8(x, torch.tensor([3, 5]), codes, scale)
    assert scale[0, 0] == 1.0 and codes[0, 0, 0, 0] == 12
    assert codes[0, 0, 3, 0] == 10 and codes[0, 0, 5, 0] == -100 and codes[0, 0, 3, 1] == 0
    assert scale[1, 0] == 0.25 and bool((codes[1] == 50).all())
    ref.store_int8(x[:1], torch.tensor([16]), codes, scale)  # offset 0: the block starts over
    assert scale[1, 0] == 0.125 and codes[1, 0, 0, 0] == 80 and bool((codes[1, 0, 1:] == 0).all())


def test_verify_oracle_by_hand():
    lg = torch.log(torch.tensor([[0.5, 0.25, 0.25], [0.2, 0.3, 0.5], [0.1, 0.1, 0.8]]))
    q = torch.tensor([[0.25, 0.5, 0.25], [0.2, 0.2, 0.6]])
    # 0.4 * 0.25 < 0.5 accepts token 0; 0.9 * 0.6 >= 0.5 refuses token 2; the residual is only token 1
    out, acc = ref.verify_drafts(lg, [0, 3], [0, 2], q, [1.0], [0.4, 0.9, 0.3], 2)
    assert out == [[0, 1, -1]] and acc == [1]
    out, acc = ref.verify_drafts(lg, [0, 3], [0, 2], None, [0.0], [0.9, 0.9, 0.3], 2)  # greedy
    assert out == [[0, 2, 2]] and acc == [2]


def test_block_copy_refusals():
    a = [torch.zeros(2, 5, 3)]
    for src, dst in (([0], [5]), ([-1], [0]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(ValueError, match="kv_copy_blocks"):
            ops.kv_copy_blocks(a, a, src, dst)


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError):
        ops.verify_drafts(torch.zeros(1, 4), torch.tensor([0, 1], dtype=torch.int32), torch.zeros(0, dtype=torch.int32),
                          None, torch.ones(1), torch.zeros(1), max_drafts=1)
    k = torch.zeros(1, 1, 16, 64, dtype=torch.int8)
    s = torch.zeros(1, 1)
    with pytest.raises(RuntimeError):
        ops.paged_attention_int8(torch.zeros(1, 1, 64, dtype=torch.bfloat16), k, k, s, s,
                                 torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), scale=1.0)


def test_draft_draws_at_any_temperature():
    """A draft model's draws: the largest logit when it is cold, nothing that raises when logits are not finite, and
    the softmax's frequencies."""
    from rlx_models_b200.runtime.speculative import SpeculativeDecoder
    sd = SpeculativeDecoder.__new__(SpeculativeDecoder)
    sd._gen, sd._draft_probs = torch.Generator().manual_seed(0), []
    x = torch.tensor([1.0, 3.0, 2.0, -float("inf")])
    for t in (1e-4, 1e-30, 1e-45, 1e-300):
        sd._temperature = t
        assert sd._pick(x) == 1 and sd._draft_probs[-1].tolist() == [0, 1, 0, 0]
    sd._temperature = 1e30
    assert sd._pick(x) != 3 and torch.allclose(sd._draft_probs[-1], torch.tensor([1, 1, 1, 0]) / 3)
    assert 0 <= sd._pick(torch.full((4,), float("nan"))) < 4
    sd._temperature, n = 1.5, 4000
    p = torch.softmax(x.double() / 1.5, 0)
    freq = torch.bincount(torch.tensor([sd._pick(x) for _ in range(n)]), minlength=4) / n
    assert bool(((freq - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all())  # five standard deviations
