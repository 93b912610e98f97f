"""Attention over int8 pages at the ends of its range: V and K scales, scores
and queries that pass fp32 or f16 on the way although the result does not."""
import pytest
import torch

from rlx_models_b200 import ops
from test_kv_int8_gpu import BF, F16_EPS, check, make_cache, make_tables, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("d", [128, 64])
def test_values_near_the_largest(cuda, d, n, sinks):
    """V scales of 2^120 (values to 2^127): whole segments, and contexts that are cut and joined."""
    g = torch.Generator().manual_seed(d + n)
    lens = [37, 200, 3000, 16]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, d, g)
    cache[3].fill_(2.0 ** 120)
    cache[3][tables[1, 3].item()] = 2.0 ** 112
    cu = [n * b for b in range(5)]
    q = (torch.randn(4 * n, 8, d, generator=g) * 0.5).to(cuda, BF)
    sk = torch.randn(8, generator=g).to(cuda) if sinks else None
    out = ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                   cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=n,
                                   scale=d ** -0.5, sinks=sk)
    ops.check_errors(cuda)
    assert bool(out.isfinite().all())
    want, mass = oracle(q, cache, tables, lens, cu, d ** -0.5, 0, sk)
    check(out, want, mass, F16_EPS)
