"""Rolling back refused drafts on int8 pages, on the host: the bookkeeping of
``SpeculativeDecoder`` over the 64-bit store and plain block copies."""
import pytest
import torch

import spec_rollback as S
from rlx_models_b200 import ops
from rlx_models_b200.ops import reference as ref


@pytest.fixture(autouse=True)
def host_ops(monkeypatch):
    def store(k, v, slots, kc, vc, ks, vs):
        ref.store_int8(k, slots, kc, ks)
        ref.store_int8(v, slots, vc, vs)

    def copy(src, dst, a, b):
        for s, d in zip(src, dst):
            d[:, list(b)] = s[:, list(a)].clone()

    monkeypatch.setattr(ops, "kv_store_int8", store)
    monkeypatch.setattr(ops, "kv_copy_blocks", copy)


@pytest.mark.parametrize("prompt_len", [5, 16, 31])
@pytest.mark.parametrize("every", [1, 2, 3, 4])
def test_refused_passes_leave_no_trace(prompt_len, every):
    S.refused_passes_leave_no_trace("cpu", prompt_len, every)


def test_without_a_roll_back_the_rows_are_coarser():
    """What the roll back is for: the scale that refused rows leave rounds the accepted ones again."""
    s = S._Seq(S.Rows("cpu"), 64)
    s.run([1, 2, 3, 4, 5], 0)
    before = {n: t.clone() for n, t in s.kv.tensors().items()}
    s.mark()
    s.run([6] + [S.WRONG] * 4, 5)
    assert bool((s.kv.k_scale[:, 0] > before["k_scale"][:, 0]).all())
    s.roll_back(5)
    for n, t in s.kv.tensors().items():
        assert bool((t[:, 0] == before[n][:, 0]).all())
    assert s.pos == 5 and s.kv.rows is None


def test_the_drafters_cache_is_rolled_back():
    sd = S.refused_passes_leave_no_trace("cpu", 9, 3)
    d = sd.draft
    # the largest of 1024 normal numbers fits 127 * 2^-4 = 7.9, that of a refused row (4 times 128) does not
    assert bool((d.kv.k_scale[:, :d.pos // 16] <= 2.0 ** -4).all())


def test_other_caches_are_left_alone():
    class Plain:
        device = torch.device("cpu")

        def make_kv_cache(self, blocks):
            self.blocks = blocks
            return object()

    m = Plain()
    s = S._Seq(m, 64)
    assert m.blocks == 5
    s.pos = 20
    s.mark()
    s.pos = 24
    s.roll_back(21)
    s.reset()
    assert s.pos == 0
