"""A branch of a running request goes on under its own parameters: the native
scheduler's stop conditions, and what ``LLMEngine.fork`` hands to it."""
import pytest
import torch

from rlx_models_b200 import _runtime
from rlx_models_b200.runtime.engine import EngineConfig, LLMEngine, RequestState, SamplingParams

EOS = 99


def staging(T=256, S=8, W=16):
    i32, i64 = torch.int32, torch.int64
    return [torch.zeros(T, dtype=i32), torch.zeros(T, dtype=i32), torch.zeros(T, dtype=i64),
            torch.zeros(S, W, dtype=i32), torch.zeros(S, dtype=i32), torch.zeros(S, W, dtype=i32),
            torch.zeros(S, dtype=i32), torch.zeros(S + 1, dtype=i32), torch.zeros(T, dtype=i64),
            torch.zeros(T, dtype=i64)]


class Host:
    """The host side of an engine: the real scheduler under ``LLMEngine.fork``, tokens chosen by the test."""

    def __init__(self, params):
        eng = self.eng = LLMEngine.__new__(LLMEngine)
        eng.cfg, eng.model, eng.stateful = EngineConfig(), object(), False
        eng.sched = _runtime.Scheduler(40, 4, 256, 16, False, 0)
        eng.kv = type("KV", (), {"copy_blocks": lambda self, src, dst: None})()
        eng.requests, eng._early, eng._inflight = {}, [], None
        eng._n_nongreedy = eng._n_host_rows = eng._n_mm = 0
        self.bufs, self.out, self.why = staging(), {}, {}
        self.a = eng.sched.add_request(list(range(20)), params.max_new_tokens, params.ignore_eos,
                                       list(params.stop_token_ids))
        eng.requests[self.a] = RequestState(self.a, 20, params, 0.0)

    def step(self, token):
        s = self.eng.sched
        info = s.schedule(*self.bufs)
        sids = self.bufs[9][:info["num_logits"]].tolist()
        for sid in sids:
            st = self.eng.requests[sid]
            st.tokens.append(token)
            if st.params.logprobs:
                st.logprobs.append(-0.5)
        for sid in s.update(sids, [token] * len(sids), EOS):
            self.out[sid], self.why[sid] = s.output_tokens(sid), s.finish_reason(sid)
        return sids


P = SamplingParams


@pytest.mark.parametrize("parent,branch,parent_ends,branch_ends", [
    (dict(ignore_eos=True), dict(ignore_eos=False), 8, 4),
    (dict(ignore_eos=False), dict(ignore_eos=True), 4, 8),
    (dict(stop_token_ids=[7]), dict(stop_token_ids=[50]), 8, 3),
    (dict(stop_token_ids=[50]), dict(stop_token_ids=[]), 3, 4),
    (dict(ignore_eos=True), dict(ignore_eos=True, max_new_tokens=2), 8, 2),
    (dict(stop_token_ids=[50]), None, 3, 3),
])
def test_branch_stops_under_its_own_parameters(parent, branch, parent_ends, branch_ends):
    """Tokens 10, 20, 50, EOS, 1, 2, 3, 4 for both. Ends are counted in tokens."""
    if parent.get("stop_token_ids") == [7]:
        parent = dict(parent, ignore_eos=False)
        parent_ends = 4
    h = Host(P(max_new_tokens=8, **parent))
    h.step(10)
    b = h.eng.fork(h.a, None if branch is None else P(**{"max_new_tokens": 8, **branch}))
    for t in (20, 50, EOS, 1, 2, 3, 4):
        h.step(t)
    assert len(h.out[h.a]) == parent_ends and len(h.out[b]) == branch_ends
    assert h.why[b] == (1 if branch_ends in (2, 8) else 2)


def test_scheduler_fork_keeps_the_parents_conditions_by_default():
    s = _runtime.Scheduler(40, 4, 256, 16, False, 0)
    bufs = staging()

    def step(tok):
        sids = bufs[9][:s.schedule(*bufs)["num_logits"]].tolist()
        return s.update(sids, [tok] * len(sids), EOS)

    a = s.add_request([1, 2, 3], 9, False, [5])
    assert step(8) == []
    b, _, _ = s.fork(a, 9)
    c, _, _ = s.fork(a, 9, ignore_eos=True)
    d, _, _ = s.fork(a, 9, stop_ids=[6])
    assert step(6) == [d]
    assert step(5) == [a, b]
    assert step(EOS) == [] and s.output_tokens(c) == [8, 6, 5, EOS]


@pytest.mark.parametrize("parent,branch", [(True, True), (True, False), (False, False)])
def test_logprobs_cover_every_token_or_none(parent, branch):
    h = Host(P(max_new_tokens=8, ignore_eos=True, logprobs=parent))
    h.step(10)
    h.step(20)
    b = h.eng.fork(h.a, P(max_new_tokens=8, ignore_eos=True, logprobs=branch))
    h.step(30)
    for sid, on in ((h.a, parent), (b, branch)):
        assert len(h.eng.requests[sid].logprobs) == (3 if on else 0)


def test_logprobs_that_the_parent_has_not_kept_are_refused():
    h = Host(P(max_new_tokens=8, ignore_eos=True))
    h.step(10)
    with pytest.raises(ValueError, match="logprobs"):
        h.eng.fork(h.a, P(max_new_tokens=8, logprobs=True))
    assert h.eng.sched.num_running() == 1
