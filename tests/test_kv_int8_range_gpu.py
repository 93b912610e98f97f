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


def far_oracle(q, cache, tables, lens, cu, scale, sinks=None):
    """64-bit attention; sum_j p_j |v_j|; sum_j p_j s_j with s_j the V scale of the key's page."""
    k, v, ks, vs = (t.cpu().double() for t in cache)
    q, tables = q.cpu().double(), tables.long()
    out, mass, unit = (torch.zeros_like(q) for _ in range(3))
    G = q.shape[1] // k.shape[1]
    for b, L in enumerate(lens):
        n, at = cu[b + 1] - cu[b], tables[b, :(L + 15) // 16]
        for h in range(q.shape[1]):
            kk = (k[at, h // G] * ks[at, h // G, None, None]).flatten(0, 1)[:L]
            vv = (v[at, h // G] * vs[at, h // G, None, None]).flatten(0, 1)[:L]
            s = q[cu[b]:cu[b + 1], h] @ kk.T * scale
            s = s.masked_fill(torch.arange(L)[None] > torch.arange(L - n, L)[:, None], -float("inf"))
            if sinks is not None:
                s = torch.cat([s, sinks[h].double().cpu().expand(n, 1)], 1)
            p = torch.softmax(s, 1)[:, :L]
            out[cu[b]:cu[b + 1], h], mass[cu[b]:cu[b + 1], h] = p @ vv, p @ vv.abs()
            unit[cu[b]:cu[b + 1], h] = (p @ vs[at, h // G].repeat_interleave(16)[:L])[:, None]
    return out, mass, unit


def far_check(got, want, mass, unit, keys):
    """As ``check`` of the other file with each key's own scale: the output's rounding; a weight's (2^-11) and its
    score's (2^-10), fp32 sums of 512 terms (2^-15), all of sum p |v|. The offset of 128 in the codes: terms of up to
    255 p s added and taken out again, 2^-22 of each: 2^-13 sum p s. Products p s below f16's normal range are off by
    up to 2^-25 where the largest of the row is at least 2^8, so by 2^-33 of it, times a code of up to 127: 2^-26 of
    sum p s for each key."""
    err = (got.cpu().double() - want).abs()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -10 + 2.0 ** -15) * mass \
        + (2.0 ** -13 + keys * 2.0 ** -26) * unit
    assert bool((err <= bound).all()), float((err / bound).max())


def leaning(cache, tables, lens, exponents, d, hq, n, g, dev):
    """V scales 2^e of the pages, and keys whose first column takes e log2 units off their scores, so that pages of all
    scales count alike. ``exponents[b][p]`` = (e, units off)."""
    for b in range(len(lens)):
        for p, (e, off) in enumerate(exponents[b]):
            at = tables[b, p].item()
            cache[3][at] = 2.0 ** e
            cache[2][at] = 2.0 ** -6
            cache[0][at, :, :, 0] = max(-127, min(127, -off))
    q = torch.randn(len(lens) * n, hq, d, generator=g) * 0.5
    q[:, :, 0] = 64.0 * 0.6875 / d ** -0.5  # one code is 0.6875 * log2(e) = 0.992 log2 units
    return q.to(dev, BF)


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("hq,d", [(8, 128), (2, 128), (16, 64)])
@pytest.mark.parametrize("kind", ["spread", "first", "middle", "last", "small first"])
def test_v_scales_far_apart(cuda, kind, hq, d, n, sinks):
    """A page whose scale is 2^60 times the others' and that has next to no weight, pages of all scales between 2^-40
    and 2^40 that count alike, and a first page of tiny values."""
    g = torch.Generator().manual_seed(hq + d + n)
    lens = [33, 250, 3001]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, d, g)
    exponents = []
    for L in lens:
        pages = (L + 15) // 16
        if kind == "spread":
            e = torch.randint(-40, 41, (pages,), generator=g).tolist()
            exponents.append([(i, i) for i in e])
        elif kind == "small first":
            exponents.append([(-70, 0)] + [(-6, 0)] * (pages - 1))
        else:
            at = {"first": 0, "middle": pages // 2, "last": pages - 1}[kind]
            exponents.append([(54, 110) if p == at else (-6, 0) for p in range(pages)])
    q = leaning(cache, tables, lens, exponents, d, hq, n, g, cuda)
    cu = [n * b for b in range(4)]
    sk = torch.randn(hq, generator=g).to(cuda) if sinks else None
    out = ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                   cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=n,
                                   scale=d ** -0.5, sinks=sk)
    ops.check_errors(cuda)
    want, mass, unit = far_oracle(q, cache, tables, lens, cu, d ** -0.5, sk)
    far_check(out, want, mass, unit, max(lens))


@pytest.mark.parametrize("power", [18, 20, 21, 24, 40])
@pytest.mark.parametrize("n", [1, 4])
def test_scores_beyond_the_spacing_of_fp32(cuda, power, n):
    """Scores of 2^24 log2 units and more, whose neighbours in fp32 lie further apart than f16's exponents reach. One
    column of q and of the keys is not zero, so scores are exact up to a factor common to the row: the largest keys of
    each row share its weight."""
    g = torch.Generator().manual_seed(power)
    lens = [40, 333, 3000]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, 128, g)
    cache[0][..., :5], cache[0][..., 6:] = 0, 0
    cache[2].fill_(1.0)
    q = torch.zeros(3 * n, 16, 128)
    q[:, :, 5] = torch.randn(3 * n, 16, generator=g) * 2.0 ** power
    q = q.to(cuda, BF)
    cu = [n * b for b in range(4)]
    out = ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                   cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=n, scale=1.0)
    ops.check_errors(cuda)
    want, mass = oracle(q, cache, tables, lens, cu, 1.0)
    check(out, want, mass, F16_EPS)


@pytest.mark.parametrize("scale", [128 ** -0.5, -0.25])
@pytest.mark.parametrize("n", [1, 3])
def test_k_scales_near_the_largest(cuda, n, scale):
    """Pages of K scale 2^120 whose products are zero (zero codes; codes only where q is zero) count as score 0, and
    one whose product is not outweighs all others or nothing. q in eighths up to 2: sums of its products with codes
    and with 128 are exact in fp32 (at most 128 * 255 * 2 = 2^16, in steps of 2^-3), as they have to be here: a
    score is off by up to 2^-13 of sum |q| times the K scale."""
    g = torch.Generator().manual_seed(n)
    lens = [100, 3000, 48]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, 128, g)
    for b, p in ((0, 2), (1, 0), (1, 100), (1, 187)):
        at = tables[b, p].item()
        cache[0][at] = 0
        cache[0][at, :, :, 7] = 3
        cache[2][at] = 2.0 ** 120
    at = tables[2, 1].item()
    cache[0][at] = 0
    cache[0][at, :, 5, 9] = 1
    cache[2][at] = 2.0 ** 120
    q = (torch.randn(3 * n, 8, 128, generator=g) * 4).round().clamp(-16, 16) / 8
    q[:, :, 7] = 0
    q[:, :4, 9], q[:, 4:, 9] = 1.0, -1.0
    q = q.to(cuda, BF)
    cu = [n * b for b in range(4)]
    out = ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                   cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=n, scale=scale)
    ops.check_errors(cuda)
    want, mass = oracle(q, cache, tables, lens, cu, scale)
    check(out, want, mass, F16_EPS)
