"""Branching a running sequence in the native scheduler: shared full blocks,
a copy of the partly filled one, independent growth, and blocks that come back."""
import pytest
import torch

from rlx_models_b200 import _runtime
from rlx_models_b200.runtime.kv_cache import PagedKVCache


def staging(T=256, S=8, W=16):
    i32, i64 = torch.int32, torch.int64
    return [torch.zeros(T, dtype=i32), torch.zeros(T, dtype=i32), torch.zeros(T, dtype=i64),
            torch.zeros(S, W, dtype=i32), torch.zeros(S, dtype=i32), torch.zeros(S, W, dtype=i32),
            torch.zeros(S, dtype=i32), torch.zeros(S + 1, dtype=i32), torch.zeros(T, dtype=i64),
            torch.zeros(T, dtype=i64)]


def step(s, bufs, token=lambda sid, i: 7):
    info = s.schedule(*bufs)
    sids = bufs[9][:info["num_logits"]].tolist()
    s.update(sids, [token(sid, i) for i, sid in enumerate(sids)], -1)
    return info, sids


@pytest.mark.parametrize("prompt", [16, 20, 31])
def test_fork_shares_full_blocks_and_copies_the_last(prompt):
    s = _runtime.Scheduler(40, 4, 256, 16, False, 0)
    bufs = staging()
    a = s.add_request(list(range(prompt)), 30, True, [])
    step(s, bufs)          # prompt
    free = s.num_free_blocks()
    b, src, dst = s.fork(a, 20)
    partly = prompt % 16 != 0
    assert (src >= 0) == partly and (dst >= 0) == partly
    assert s.num_free_blocks() == free - int(partly)
    info, sids = step(s, bufs, lambda sid, i: 100 + sid)
    assert info["num_decode"] == 2 and set(sids) == {a, b}
    tables = {sid: bufs[3][i].tolist() for i, sid in enumerate(sids)}
    full = prompt // 16
    assert tables[a][:full] == tables[b][:full]
    assert tables[a][full] != tables[b][full]       # each writes a block of its own
    if partly:
        assert tables[a][full] == src and tables[b][full] == dst
    while s.has_work():
        step(s, bufs, lambda sid, i: 100 + sid)
    assert s.output_tokens(a)[0] == s.output_tokens(b)[0] == 7
    assert s.output_tokens(a)[1:] == [100 + a] * 29 and s.output_tokens(b)[1:] == [100 + b] * 19
    assert s.num_free_blocks() == 40


def test_a_fork_outlives_its_parent_and_a_preemption():
    s = _runtime.Scheduler(8, 4, 256, 16, True, 0)
    bufs = staging()
    a = s.add_request(list(range(40)), 60, True, [])
    step(s, bufs)
    b, _, _ = s.fork(a, 60)
    s.abort(a)
    while s.has_work():
        step(s, bufs)
    assert len(s.output_tokens(b)) == 60
    c = s.add_request(list(range(1, 30)), 40, True, [])
    step(s, bufs)
    d, _, _ = s.fork(c, 70)  # together they need more than the 8 blocks: one is preempted and recomputed
    while s.has_work():
        step(s, bufs)
    assert len(s.output_tokens(c)) == 40 and len(s.output_tokens(d)) == 70
    assert s.stats()["preemptions"] >= 1 and s.num_free_blocks() == 8


def test_fork_refusals():
    s = _runtime.Scheduler(3, 2, 256, 16, False, 0)
    bufs = staging()
    a = s.add_request(list(range(20)), 12, True, [])
    with pytest.raises(ValueError, match="not decoding"):
        s.fork(a, 12)  # still waiting
    step(s, bufs)
    for bad in (1, 0, 10 ** 6):
        with pytest.raises(ValueError):
            s.fork(a, bad)  # reached already, and longer than the context
    with pytest.raises(ValueError, match="not decoding"):
        s.fork(a + 5, 12)
    s.fork(a, 12)
    with pytest.raises(RuntimeError, match="max_num_seqs"):
        s.fork(a, 12)
    s2 = _runtime.Scheduler(2, 4, 256, 16, False, 0)
    c = s2.add_request(list(range(20)), 2, True, [])
    step(s2, bufs)
    with pytest.raises(RuntimeError, match="no free KV block"):
        s2.fork(c, 2)


def test_int8_cache_layout_and_refusals():
    kv = PagedKVCache(2, 3, 4, 64, device="cpu", dtype=torch.int8)
    assert list(kv.tensors()) == ["k", "v", "k_scale", "v_scale"]
    assert kv.k.shape == (2, 3, 4, 16, 64) and kv.k_scale.shape == (2, 3, 4)
    held = sum(t.numel() * t.element_size() for t in kv.tensors().values())
    assert held == 3 * PagedKVCache.bytes_per_block(2, 4, 64, 1, 4)
    with pytest.raises(ValueError, match="head_dim"):
        PagedKVCache(1, 1, 1, 256, device="cpu", dtype=torch.int8)
    with pytest.raises(ValueError, match="dtype"):
        PagedKVCache(1, 1, 1, 64, device="cpu", dtype=torch.int16)
    with pytest.raises(ValueError, match="KV blocks hold"):
        kv.scatter_blocks({"k": kv.k, "v": kv.v}, [0], [1])
