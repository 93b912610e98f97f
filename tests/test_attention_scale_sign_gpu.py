"""Softmax scales of zero and below, for a prefill over bf16 pages and for
attention over int8 pages read directly and through bf16 copies."""
import pytest
import torch

from rlx_models_b200 import ops
import test_kv_int8_gpu as I
import test_prefill_tiles_gpu as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [-0.09, 0.0])
@pytest.mark.parametrize("window,causal", [(0, True), (50, True), (0, False)])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (32, 8)])
def test_prefill(cuda, hq, hkv, window, causal, scale):
    g = torch.Generator().manual_seed(hq)
    lens, n = [700, 33, 300, 0], [500, 33, 257, 3]
    if not causal:
        lens, n = [700, 130], [700, 130]
    q, k, v, tables, ctx, cu = P.make(cuda, lens, n, hq, hkv, g)
    got = ops.prefill_attention(q, k, v, tables, ctx, torch.tensor(cu, dtype=torch.int32, device=cuda), max(n),
                                scale=scale, window=window, causal=causal)
    ops.check_errors(cuda)
    P.check(got, q, k, v, tables, lens, cu, scale, window, None, causal)


@pytest.mark.parametrize("scale", [-0.09, 0.0])
@pytest.mark.parametrize("n", [1, 3, 130])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(0, False), (20, True)])
def test_int8_pages(cuda, hq, hkv, d, n, window, sinks, scale):
    g = torch.Generator().manual_seed(n + hq)
    lens = [400, 0, 131, 1000]
    tables, nb = I.make_tables(lens, g)
    cache = I.make_cache(cuda, nb, hkv, d, g)
    cu = [n * b for b in range(5)]
    sk = torch.randn(hq, generator=g).to(cuda) if sinks else None
    q = (torch.randn(4 * n, hq, d, generator=g) * 0.5).to(cuda, I.BF)
    out = ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                   cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=n, scale=scale,
                                   window=window, sinks=sk)
    ops.check_errors(cuda)
    want, mass = I.oracle(q, cache, tables, lens, cu, scale, window, sk)
    I.check(out, want, mass, I.weight_eps(hq, hkv, n, d))
