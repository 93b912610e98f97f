"""Rolling back refused drafts on int8 pages: given rows (four times the size
where a draft is refused), and a served model's own."""
import pytest
import torch

import spec_rollback as S
from rlx_models_b200 import config as C, ops
from rlx_models_b200.ops import reference as ref
from rlx_models_b200.registry import build_model
from rlx_models_b200.runtime.speculative import _Seq

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompt_len", [5, 16, 31])
@pytest.mark.parametrize("every", [1, 2, 3, 4])
def test_refused_passes_leave_no_trace(cuda, prompt_len, every):
    S.refused_passes_leave_no_trace(cuda, prompt_len, every)
    ops.check_errors(cuda)


@pytest.mark.parametrize("accepted", [0, 1, 3, 5])
@pytest.mark.parametrize("prompt_len", [13, 32])
def test_a_models_rows(cuda, prompt_len, accepted):
    model = build_model(C.tiny(), device=cuda, seed=0)
    model.set_kv_cache_dtype("int8")
    s = _Seq(model, 128)
    s.run(list(range(prompt_len)), 0)
    want = {n: t.cpu().clone() for n, t in s.kv.tensors().items()}
    s.mark()
    s.run([9, 8, 7, 6, 5], prompt_len)
    rows = [(k.cpu(), v.cpu()) for k, v in s.kv.rows]
    s.roll_back(prompt_len + accepted)
    ops.check_errors(cuda)
    assert s.pos == prompt_len + accepted
    for layer, (k, v) in enumerate(rows):
        for t in range(accepted):
            at = torch.tensor([prompt_len + t])
            ref.store_int8(k[t:t + 1], at, want["k"][layer], want["k_scale"][layer])
            ref.store_int8(v[t:t + 1], at, want["v"][layer], want["v_scale"][layer])
    blocks = (prompt_len + accepted + 15) // 16
    for n, t in s.kv.tensors().items():
        assert bool((t[:, :blocks].cpu() == want[n][:, :blocks]).all()), n
