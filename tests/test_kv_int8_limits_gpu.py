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


@pytest.mark.parametrize("hq,d", [(8, 128), (8, 64)])  # by copies when long, directly
@pytest.mark.parametrize("cu", [[0, 60, 400], [0, 200, 201], [-7, 60, 120], [0, 90, 30], [130, 140, 150]])
def test_offsets_outside_the_queries(cuda, hq, d, cu):
    """``cu_q`` that leaves q's 120 rows: an error, and no row outside ``out`` is written."""
    g = torch.Generator().manual_seed(18)
    tables, nb = make_tables([410, 410], g)
    cache = make_cache(cuda, nb, 2, d, g)
    room = torch.full((720, hq, d), 7.0, dtype=BF, device=cuda)
    out = room[300:420]
    q = torch.randn(120, hq, d, generator=g).to(cuda, BF)
    for most in (5, 300):
        ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor([410, 410], dtype=torch.int32, device=cuda),
                                 cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=most, scale=0.1,
                                 out=out)
        with pytest.raises(ops.KernelError, match="bounds"):
            ops.check_errors(cuda)
    assert bool((room[:300] == 7.0).all()) and bool((room[420:] == 7.0).all())


def test_the_last_rows_of_the_queries(cuda):
    """Offsets up to the last row are in order, an empty sequence at the end among them."""
    g = torch.Generator().manual_seed(19)
    tables, nb = make_tables([50, 410, 3], g)
    cache = make_cache(cuda, nb, 2, 128, g)
    q = torch.randn(120, 8, 128, generator=g).to(cuda, BF)
    ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor([50, 410, 3], dtype=torch.int32, device=cuda),
                             cu_q=torch.tensor([0, 20, 120, 120], dtype=torch.int32, device=cuda), max_q_len=100,
                             scale=0.1)
    ops.check_errors(cuda)
