"""Prefill attention with one and with two query tiles a CTA (large batches):
against the 64-bit definition, and bit for bit against each other, for odd
numbers of tiles, windows in which the two tiles of a CTA begin and end apart,
sinks, rows without keys and garbage behind the contexts."""
import math

import pytest
import torch

from rlx_models_b200 import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def make(dev, lens, n, hq, hkv, g):
    pages = [max((l + 15) // 16, 1) for l in lens]
    k, v = (torch.randn(sum(pages) + 1, hkv, 16, 128, generator=g).to(dev, BF) for _ in range(2))
    perm = torch.randperm(sum(pages), generator=g).int()
    tables = torch.full((len(lens), max(pages)), sum(pages), dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        tables[b, :p] = perm[at:at + p]
        at += p
    cu = [0]
    for i in n:
        cu.append(cu[-1] + i)
    q = torch.randn(cu[-1], hq, 128, generator=g).to(dev, BF)
    return q, k, v, tables.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), cu


def check(got, q, k, v, tables, lens, cu, scale, window, sinks, causal=True):
    """P is rounded to bf16 (half a step: 2^-8 of each weight), then the output (2^-8 of it); fp32 scores and sums of
    128 products and of a row stay below 2^-13 of the mass sum_j p_j |v_j|."""
    G = q.shape[1] // k.shape[1]
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        o = got[cu[b]:cu[b + 1]].double()
        if n == 0 or L == 0:
            assert not bool(o.any())
            continue
        at = tables[b, :(L + 15) // 16].long()
        kk, vv = (t[at].transpose(0, 1).flatten(1, 2)[:, :L].double().repeat_interleave(G, 0) for t in (k, v))
        s = (q[cu[b]:cu[b + 1]].double().transpose(0, 1) @ kk.transpose(1, 2)) * scale
        pos = torch.arange(L - n, L, device=q.device)[:, None]
        j = torch.arange(L, device=q.device)[None]
        hide = (j > pos) if causal else torch.zeros_like(j > pos)
        if window:
            hide = hide | (j <= pos - window)
        s = s.masked_fill(hide, -math.inf)
        if sinks is not None:
            s = torch.cat([s, sinks.double()[:, None, None].expand(-1, n, 1)], 2)
        p = torch.nan_to_num(torch.softmax(s, 2))[:, :, :L]
        want, mass = (p @ vv).transpose(0, 1), (p @ vv.abs()).transpose(0, 1)
        bound = (2.0 ** -8 + 2.0 ** -13) * mass + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -7)
        assert bool(((o - want).abs() <= bound).all()), (b, ((o - want).abs() - bound).max())


@pytest.mark.parametrize("hq,hkv", [(32, 8), (64, 8), (16, 16)])
@pytest.mark.parametrize("window,with_sinks", [(0, False), (0, True), (40, False), (200, True), (1, False)])
def test_two_tiles_a_cta(cuda, hq, hkv, window, with_sinks):
    g = torch.Generator().manual_seed(hq + window)
    lens, n = [900, 33, 300, 1, 20, 0, 640], [700, 33, 257, 1, 50, 3, 31]  # 50 queries over 20 keys: 30 see nothing
    q, k, v, tables, ctx, cu = make(cuda, lens, n, hq, hkv, g)
    sinks = torch.randn(hq, generator=g).to(cuda) if with_sinks else None
    scale = 128 ** -0.5
    kw = dict(scale=scale, window=window, sinks=sinks)
    got = ops.prefill_attention(q, k, v, tables, ctx, torch.tensor(cu, dtype=torch.int32, device=cuda), max(n), **kw)
    ops.check_errors(cuda)
    check(got, q, k, v, tables, lens, cu, scale, window, sinks)
    # one sequence and one KV head at a time: one tile a CTA
    G = hq // hkv
    for b in range(len(lens)):
        for h in (0, hkv - 1):
            s = sinks[h * G:h * G + G].contiguous() if with_sinks else None
            one = ops.prefill_attention(
                q[cu[b]:cu[b + 1], h * G:h * G + G].contiguous(), k[:, h:h + 1].contiguous(),
                v[:, h:h + 1].contiguous(), tables[b:b + 1], ctx[b:b + 1],
                torch.tensor([0, n[b]], dtype=torch.int32, device=cuda), n[b], scale=scale, window=window, sinks=s)
            assert torch.equal(one, got[cu[b]:cu[b + 1], h * G:h * G + G])
    ops.check_errors(cuda)


def test_two_tiles_not_causal(cuda):
    g = torch.Generator().manual_seed(3)
    lens, n = [700, 130, 400], [700, 130, 400]
    q, k, v, tables, ctx, cu = make(cuda, lens, n, 24, 24, g)
    got = ops.prefill_attention(q, k, v, tables, ctx, torch.tensor(cu, dtype=torch.int32, device=cuda), 700, scale=0.09,
                                causal=False)
    ops.check_errors(cuda)
    check(got, q, k, v, tables, lens, cu, 0.09, 0, None, causal=False)


def test_two_tiles_from_int8_pages(cuda):
    """A chunk over int8 pages (their copies lie in order) in CTAs of two tiles; the pages behind a context are NaN."""
    g = torch.Generator().manual_seed(4)
    lens, n, hq, hkv = [1000, 77, 513], [600, 77, 300], 32, 8
    q, k, v, tables, ctx, cu = make(cuda, lens, n, hq, hkv, g)
    codes = [torch.randint(-127, 128, k.shape, generator=g, dtype=torch.int8).to(cuda) for _ in range(2)]
    sc = [torch.full(k.shape[:2], 2.0 ** -6, device=cuda) for _ in range(2)]
    wide = [(c.double() * 2.0 ** -6).to(BF) for c in codes]
    for t in sc:
        t[-1] = float("nan")  # the block that tables hold behind the contexts
    cu_q = torch.tensor(cu, dtype=torch.int32, device=cuda)
    got = ops.paged_attention_int8(q, *codes, *sc, tables, ctx, cu_q=cu_q, max_q_len=600, scale=0.09, window=333)
    ops.check_errors(cuda)
    check(got, q, *wide, tables, lens, cu, 0.09, 333, None)
    same = ops.prefill_attention(q, *wide, tables, ctx, cu_q, 600, scale=0.09, window=333)
    assert torch.equal(got, same)


def test_two_tiles_in_a_graph_on_another_stream(cuda):
    g = torch.Generator().manual_seed(5)
    lens, n = [1024] * 4, [512] * 4
    q, k, v, tables, ctx, cu = make(cuda, lens, n, 32, 8, g)
    cu_q = torch.tensor(cu, dtype=torch.int32, device=cuda)
    want = ops.prefill_attention(q, k, v, tables, ctx, cu_q, 512, scale=0.09)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            ops.prefill_attention(q, k, v, tables, ctx, cu_q, 512, scale=0.09, out=out)
        for _ in range(3):
            out.zero_()
            graph.replay()
    side.synchronize()
    assert torch.equal(out, want)
    ops.check_errors(cuda)


@pytest.mark.parametrize("window", [0, 48, 500])
def test_second_tile_empty_or_apart(cuda, window):
    """CTAs whose second tile has no tokens, or begins behind the first one's keys, many at once and again and again:
    the thread that issues its products must neither miss a turn nor hold up the loads."""
    g = torch.Generator().manual_seed(6)
    n = [32] * 40 + [64] * 4 + [33, 1, 96, 128] * 4
    lens = [l + 1400 for l in n]
    q, k, v, tables, ctx, cu = make(cuda, lens, n, 32, 8, g)
    cu_q = torch.tensor(cu, dtype=torch.int32, device=cuda)
    want = ops.prefill_attention(q, k, v, tables, ctx, cu_q, 128, scale=0.09, window=window)
    check(want, q, k, v, tables, lens, cu, 0.09, window, None)
    out = torch.empty_like(q)
    for _ in range(60):
        ops.prefill_attention(q, k, v, tables, ctx, cu_q, 128, scale=0.09, window=window, out=out)
        assert torch.equal(out, want)
    ops.check_errors(cuda)
