"""Arguments of attention over int8 pages that do not fit, read directly and
through bf16 copies: reported, and nothing outside the outputs is touched."""
import pytest
import torch

from rlx_models_b200 import ops
from test_kv_int8_gpu import BF, make_cache, make_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,most", [(3, 2), (200, 100), (200, 199), (300, 20)])
def test_more_queries_than_announced(cuda, n, most):
    g = torch.Generator().manual_seed(17)
    lens = [310, 310]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, 128, g)
    q = torch.randn(n + 1, 8, 128, generator=g).to(cuda, BF)
    args = (q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda))
    cu = torch.tensor([0, 1, n + 1], dtype=torch.int32, device=cuda)
    ops.paged_attention_int8(*args, cu_q=cu, max_q_len=n, scale=0.1)
    ops.check_errors(cuda)
    ops.paged_attention_int8(*args, cu_q=cu, max_q_len=most, scale=0.1)
    with pytest.raises(ops.KernelError, match="bounds"):
        ops.check_errors(cuda)
