"""int8 paged KV cache with power-of-two block scales: the store (bit-exact
against the 64-bit definition), the bf16 page copies (exact), attention over
the pages (decode, multi-token verification, chunks; windows, sinks, softcap,
empty rows, garbage behind the contexts), block copies, and their use on other
streams, in graphs and at large offsets."""
import math

import pytest
import torch

from rlx_models_b200 import ops
from rlx_models_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def make_cache(dev, nb, hkv, d, g):
    codes = torch.randint(-127, 128, (2, nb, hkv, 16, d), generator=g, dtype=torch.int8)
    scale = torch.ldexp(torch.ones(2, nb, hkv), torch.randint(-9, -3, (2, nb, hkv), generator=g))
    return [t.contiguous().to(dev) for t in (codes[0], codes[1], scale[0], scale[1])]


def make_tables(lens, g, extra=3):
    pages = [(l + 15) // 16 for l in lens]
    nb = sum(pages) + extra
    perm = torch.randperm(nb, generator=g)
    tables = torch.full((len(lens), max(max(pages), 1)), nb - 1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        tables[b, :n] = perm[at:at + n].int()
        at += n
    return tables, nb


def oracle(q, cache, tables, lens, cu, scale, window=0, sinks=None, softcap=0.0):
    """64-bit attention and, per output, what its error is bounded by, see ``check``: (sum_j p_j |v_j|
    + 2^-22 sum_j |v_j|, the largest V scale among the pages)."""
    k, v, ks, vs = (t.cpu().double() for t in cache)
    q, tables = q.cpu().double(), tables.cpu().long()
    out, mass, top = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    G = q.shape[1] // k.shape[1]
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0 or L == 0:
            continue
        at = tables[b, :(L + 15) // 16]
        kk = (k[at] * ks[at][:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :L]
        vv = (v[at] * vs[at][:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :L]
        pos = torch.arange(L - n, L)[:, None]
        j = torch.arange(L)[None]
        hide = j > pos
        if window:
            hide |= j <= pos - window
        for h in range(q.shape[1]):
            s = q[cu[b]:cu[b + 1], h] @ kk[h // G].T * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            s = s.masked_fill(hide, -math.inf)
            if sinks is not None:
                s = torch.cat([s, sinks[h].double().cpu().expand(n, 1)], 1)
            p = torch.nan_to_num(torch.softmax(s, 1))[:, :L]
            out[cu[b]:cu[b + 1], h] = p @ vv[h // G]
            seen = (~hide).double()
            mass[cu[b]:cu[b + 1], h] = p @ vv[h // G].abs() + 2.0 ** -22 * (seen @ vv[h // G].abs())
            top[cu[b]:cu[b + 1], h] = vs[at, h // G].max()
    return out, (mass, top)


def check(out, want, mass, weight_eps):
    """Output rounding: half a step of bf16 (2^-8). Each weight is rounded to 16 bits (half a step:
    ``weight_eps``) and its score carries fp32 rounding: scores stay below 2^6 here, so products summed
    in fp32 (2^-24 each, at most 128 + a few) and ex2 (2^-22) move a weight by less than 2^-10 of it at the
    very most; they enter as sum_j p_j |v_j|. Sums of l and of O are fp32: 2^-15 covers 512 of them. Below f16's normal
    range a weight is off by up to half its smallest step, 2^-25, where the largest weight of a row is at least
    2^8: 2^-33 |v_j| for each key, and weight_eps * 2^-22 = 2^-33. V enters its products as code + 128 and a
    second product takes 128 sum p out again, page by page: the two add terms of up to 255 s p of the page to an
    fp32 sum, each with an error of at most 2^-22 of them (tensor cores may truncate): over all pages, whose p add
    up to 1, at most 2 * 2^-22 * 255 s < 2^-13 s with s the largest scale."""
    mass, top = mass
    err = (out.cpu().double() - want).abs()
    bound = 2.0 ** -8 * want.abs() + (weight_eps + 2.0 ** -10 + 2.0 ** -15) * mass + 2.0 ** -13 * top + 1e-30
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0


F16_EPS, BF16_EPS = 2.0 ** -11, 2.0 ** -8


def weight_eps(hq, hkv, n, d=128):
    """Pages read directly: weights in f16. Through bf16 copies: ``prefill_attention`` rounds them to bf16."""
    copies = n * hq > ops.INT8_DIRECT_ROWS * hkv and d == 128 and 8 * hkv % hq == 0
    return BF16_EPS if copies else F16_EPS

DECODE = [1, 15, 16, 17, 100, 513, 2047]


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (64, 8, 64), (8, 8, 128), (5, 1, 64), (14, 2, 128), (16, 1, 128),
                                      (16, 1, 64), (6, 2, 64)])
@pytest.mark.parametrize("window,sinks,cap", [(0, False, 0.0), (128, True, 0.0), (37, False, 0.0), (0, True, 20.0)])
def test_decode(cuda, hq, hkv, d, window, sinks, cap):
    g = torch.Generator().manual_seed(hq * d + window)
    tables, nb = make_tables(DECODE, g)
    cache = make_cache(cuda, nb, hkv, d, g)
    q = (torch.randn(len(DECODE), hq, d, generator=g) * 0.5).to(cuda, BF)
    sk = torch.randn(hq, generator=g).to(cuda) if sinks else None
    ctx = torch.tensor(DECODE, dtype=torch.int32, device=cuda)
    out = ops.paged_attention_int8(q, *cache, tables.to(cuda), ctx, scale=d ** -0.5, window=window, sinks=sk,
                                   softcap=cap)
    ops.check_errors(cuda)
    want, mass = oracle(q, cache, tables, DECODE, list(range(len(DECODE) + 1)), d ** -0.5, window, sk, cap)
    check(out, want, mass, F16_EPS)


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (64, 8, 64), (7, 1, 128), (16, 1, 64), (3, 3, 64)])
@pytest.mark.parametrize("new", [[1, 5, 3, 2, 4], [8, 0, 7, 1, 8], [2, 2, 2, 2, 2]])
@pytest.mark.parametrize("window", [0, 20])
def test_several_queries(cuda, hq, hkv, d, new, window):
    lens = [1, 40, 3, 700, 33]
    lens = [max(l, n) for l, n in zip(lens, new)]
    g = torch.Generator().manual_seed(hq + sum(new))
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, hkv, d, g)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = (torch.randn(cu[-1] + 2, hq, d, generator=g) * 0.5).to(cuda, BF)
    out = torch.full_like(q, 7.0)  # two rows behind the last sequence keep this
    ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                             cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=max(new),
                             scale=d ** -0.5, window=window, out=out)
    ops.check_errors(cuda)
    want, mass = oracle(q[:cu[-1]], cache, tables, lens, cu, d ** -0.5, window)
    check(out[:cu[-1]], want, mass, weight_eps(hq, hkv, max(new), d))
    assert bool((out[cu[-1]:] == 7.0).all())


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (64, 8, 64), (6, 2, 64), (3, 1, 128), (16, 1, 128)])
@pytest.mark.parametrize("window,sinks,cap", [(0, False, 0.0), (20, True, 0.0), (128, False, 0.0), (0, True, 15.0)])
def test_chunks(cuda, hq, hkv, d, window, sinks, cap):
    lens, new = [300, 129, 77], [130, 129, 1]
    g = torch.Generator().manual_seed(5)
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, hkv, d, g)
    cu = [0, 130, 259, 260]
    sk = torch.randn(hq, generator=g).to(cuda) if sinks else None
    q = (torch.randn(260, hq, d, generator=g) * 0.5).to(cuda, BF)
    out = ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                   cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=130,
                                   scale=d ** -0.5, window=window, sinks=sk, softcap=cap)
    ops.check_errors(cuda)
    want, mass = oracle(q, cache, tables, lens, cu, d ** -0.5, window, sk, cap)
    check(out, want, mass, F16_EPS if cap else weight_eps(hq, hkv, 130, d))


def test_chunks_in_groups(cuda, monkeypatch):
    """Wide block tables: the bf16 copies are made for a few sequences at a time."""
    lens, new = [300, 0, 129, 77], [130, 0, 129, 40]
    g = torch.Generator().manual_seed(6)
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, 128, g)
    cu = [0, 130, 130, 259, 299]
    q = (torch.randn(299, 8, 128, generator=g) * 0.5).to(cuda, BF)
    args = (q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda))
    kw = dict(cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=130, scale=0.1)
    whole = ops.paged_attention_int8(*args, **kw)
    for limit in (1, 400000):
        monkeypatch.setattr(ops, "INT8_COPY_BYTES", limit)
        assert torch.equal(whole, ops.paged_attention_int8(*args, **kw))
    ops.check_errors(cuda)


def test_what_does_not_fit_is_reported(cuda):
    """Contexts longer than the block table and more queries than ``max_q_len``."""
    g = torch.Generator().manual_seed(17)
    tables, nb = make_tables([40, 40], g)
    cache = make_cache(cuda, nb, 2, 128, g)
    for n, most, ctx in ((1, 1, 49), (3, 2, 40), (40, 40, 400)):
        q = torch.randn(2 * n, 8, 128, generator=g).to(cuda, BF)
        ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor([40, ctx], dtype=torch.int32, device=cuda),
                                 cu_q=torch.tensor([0, n, 2 * n], dtype=torch.int32, device=cuda), max_q_len=most,
                                 scale=0.1)
        with pytest.raises(ops.KernelError, match="bounds"):
            ops.check_errors(cuda)


@pytest.mark.parametrize("n", [1, 3, 40])
def test_rows_without_keys(cuda, n):
    """Contexts of length zero, and more queries than keys: the rows in front of the first key give 0."""
    g = torch.Generator().manual_seed(1)
    lens = [0, 2, 0, 50]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 8, 128, g)
    cu = [0, n, 2 * n, 3 * n, 4 * n]
    q = torch.randn(4 * n, 32, 128, generator=g).to(cuda, BF)
    for sinks in (None, torch.zeros(32, device=cuda)):
        out = ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                       cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_q_len=n,
                                       scale=0.1, sinks=sinks)
        ops.check_errors(cuda)
        want, mass = oracle(q, cache, tables, lens, cu, 0.1, sinks=sinks)
        check(out, want, mass, weight_eps(32, 8, n))
        assert bool((out[:n] == 0).all()) and bool((out[2 * n:3 * n] == 0).all())


def test_long_contexts_split(cuda):
    """Contexts much longer than others, cut over many CTAs, and more sequences than threads of a CTA."""
    g = torch.Generator().manual_seed(2)
    lens = [20000, 1, 3001] + [5] * 150
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, 128, g)
    q = torch.randn(len(lens), 8, 128, generator=g).to(cuda, BF)
    out = ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                   scale=0.05)
    ops.check_errors(cuda)
    want, mass = oracle(q, cache, tables, lens, list(range(len(lens) + 1)), 0.05)
    check(out, want, mass, F16_EPS)


def test_scales_far_apart_and_large_queries(cuda):
    """V scales that grow along the context, tiny ones first, and queries outside f16's range."""
    g = torch.Generator().manual_seed(3)
    lens = [200, 200]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 1, 128, g)
    for p in range(13):
        for b in range(2):
            cache[3][tables[b, p].item()] = 2.0 ** (-20 + p) if b == 0 else 2.0 ** (8 - p)
    cache[2].fill_(2.0 ** -24)
    q = (torch.randn(2, 4, 128, generator=g) * 2.0 ** 20).to(cuda, BF)
    out = ops.paged_attention_int8(q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                   scale=2.0 ** -7)
    ops.check_errors(cuda)
    want, mass = oracle(q, cache, tables, lens, [0, 1, 2], 2.0 ** -7)
    check(out, want, mass, F16_EPS)


def test_garbage_behind_the_context(cuda):
    """NaN scales of blocks that no context reaches and any code behind the last token change nothing."""
    g = torch.Generator().manual_seed(4)
    lens = [33, 16]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, 64, g)
    used = set(tables[0, :3].tolist() + tables[1, :1].tolist())
    q = torch.randn(2, 4, 64, generator=g).to(cuda, BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda)
    a = ops.paged_attention_int8(q, *cache, tables.to(cuda), ctx, scale=0.1)
    other = [t.clone() for t in cache]
    for b in range(nb):
        if b not in used:
            other[2][b] = other[3][b] = float("nan")
    last = tables[0, 2].item()
    other[0][last, :, 1:], other[1][last, :, 1:] = 127, -128
    b = ops.paged_attention_int8(q, *other, tables.to(cuda), ctx, scale=0.1)
    assert torch.equal(a, b)


def test_nan_query_stays_in_its_row(cuda):
    g = torch.Generator().manual_seed(4)
    lens = [33, 160]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, 64, g)
    q = torch.randn(2, 4, 64, generator=g).to(cuda, BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda)
    a = ops.paged_attention_int8(q, *cache, tables.to(cuda), ctx, scale=0.1)
    q[1, 1, 5] = float("nan")
    b = ops.paged_attention_int8(q, *cache, tables.to(cuda), ctx, scale=0.1)
    assert bool(b[1, 1].isnan().all())
    keep = torch.ones(2, 4, dtype=torch.bool, device=cuda)
    keep[1, 1] = False
    assert torch.equal(a[keep], b[keep])


@pytest.mark.parametrize("d,hkv", [(128, 8), (64, 3), (128, 1)])
def test_store_is_exact(cuda, d, hkv):
    """A prefill over several blocks, then tokens one by one that grow and do not grow the scales."""
    g = torch.Generator().manual_seed(d)
    nb = 9
    cache = make_cache(cuda, nb, hkv, d, g)
    want = [t.cpu().clone() for t in cache]

    def put(slots, x, y):
        s = torch.tensor(slots, dtype=torch.int64)
        ops.kv_store_int8(x.to(cuda), y.to(cuda), s.to(cuda), *cache)
        ops.check_errors(cuda)
        ref.store_int8(x, s, want[0], want[2])
        ref.store_int8(y, s, want[1], want[3])
        for got, w in zip(cache, want):
            assert torch.equal(got.cpu(), w)

    def rnd(n, f=1.0):
        return ((torch.randn(n, hkv, d, generator=g) * f).to(BF), (torch.randn(n, hkv, d, generator=g) * f).to(BF))

    put(list(range(3 * 16, 3 * 16 + 37)) + [7 * 16 + o for o in range(5, 16)], *rnd(48))
    for i, f in enumerate((1.0, 0.1, 40.0, 3.0, 1e-6, 5000.0)):
        put([5 * 16 + 5 + i, 7 * 16 + i], *rnd(2, f))
    put([-1, 2 * 16 + 3, 2 * 16 + 4, 2 * 16 + 3, -5], *rnd(5))  # skipped rows, and a slot that comes twice
    put([4 * 16] * 40 + [-1], *rnd(41))                        # padding rows of one slot
    x, y = rnd(2, 0.0)
    put([6 * 16, 6 * 16 + 1], x, y)                            # zeros only
    x, y = rnd(3)
    x[0, 0, 0], x[1, 0, 1], y[2, 0, 2], y[0, 0, 3] = float("nan"), float("inf"), -float("inf"), 3e38
    put([16, 17, 18], x, y)
    x, y = rnd(16)
    x[:, :, 0] = 127.0 / 64  # the largest magnitude that a scale holds, and the next bf16 value above it
    y[:, :, 0] = 255.0 / 128
    put(list(range(16)), x, y)


def test_store_infinity_beside_the_largest_value(cuda):
    """127 times the scale of bf16's largest value passes fp32: an infinity next to it is still +-127 steps."""
    top = torch.finfo(BF).max
    x = torch.zeros(2, 2, 64, dtype=BF)
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 2], x[0, 0, 3], x[1, 0, 4] = top, float("inf"), -float("inf"), -top, float("nan")
    x[1, 1, 0], x[1, 1, 1] = -top, 1.0
    slots = torch.tensor([16, 17])
    cache = make_cache(cuda, 2, 2, 64, torch.Generator().manual_seed(0))
    want = [t.cpu() for t in cache]
    ops.kv_store_int8(x.to(cuda), x.to(cuda), slots.to(cuda), *cache)
    for i in (0, 1):
        ref.store_int8(x, slots, want[i], want[2 + i])
    assert want[0][1, 0, 0, :4].tolist() == [64, 127, -127, -64]
    for got, w in zip(cache, want):
        assert torch.equal(got.cpu(), w)


def test_store_reads_strided_rows(cuda):
    g = torch.Generator().manual_seed(8)
    fused = torch.randn(20, 12, 128, generator=g).to(cuda, BF)
    slots = torch.arange(20, device=cuda) + 16
    a, b = make_cache(cuda, 4, 2, 128, g), None
    b = [t.clone() for t in a]
    ops.kv_store_int8(fused[:, 8:10], fused[:, 10:], slots, *a)
    ops.kv_store_int8(fused[:, 8:10].contiguous(), fused[:, 10:].contiguous(), slots, *b)
    c = [t.clone() for t in b]
    odd = torch.randn(20, 2 * 128 + 1, generator=g).to(cuda, BF)[:, 1:].view(20, 2, 128)  # not 16-byte aligned
    ops.kv_store_int8(odd, odd, slots, *c)
    ops.kv_store_int8(odd.contiguous(), odd.contiguous(), slots, *b)
    ops.check_errors(cuda)
    assert all(torch.equal(x, y) for x, y in zip(b, c))
    ops.kv_store_int8(fused[:, 8:10], fused[:, 10:], slots, *b)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_store_long_batch(cuda):
    """More than 1024 tokens: warps take groups of 16, runs cross the groups."""
    g = torch.Generator().manual_seed(9)
    T = 1501
    cache = make_cache(cuda, 101, 2, 64, g)
    want = [t.cpu().clone() for t in cache]
    x, y = torch.randn(T, 2, 64, generator=g).to(BF), torch.randn(T, 2, 64, generator=g).to(BF)
    slots = torch.cat([torch.arange(700) + 5, torch.arange(801) + 720])
    ops.kv_store_int8(x.to(cuda), y.to(cuda), slots.to(cuda), *cache)
    ops.check_errors(cuda)
    ref.store_int8(x, slots, want[0], want[2])
    ref.store_int8(y, slots, want[1], want[3])
    for got, w in zip(cache, want):
        assert torch.equal(got.cpu(), w)


def test_page_copies_are_exact(cuda):
    g = torch.Generator().manual_seed(10)
    lens = [40, 0, 16]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 3, 64, g)
    k, v, t = ops.kv_dequant_pages_int8(*cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda))
    ops.check_errors(cuda)
    assert t.tolist() == [[0, 1, 2], [3, 4, 5], [6, 7, 8]]
    for b, l in enumerate(lens):
        for p in range((l + 15) // 16):
            at = tables[b, p].item()
            for got, c, s in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
                assert torch.equal(got[t[b, p]].double(), c[at].double() * s[at].double()[:, None, None])
    assert bool((k[3] == 0).all()) and bool((v[3] == 0).all())


def test_unknown_blocks_are_reported(cuda):
    """A block id outside the cache is an error at the next check, not an access outside it."""
    g = torch.Generator().manual_seed(11)
    cache = make_cache(cuda, 4, 2, 64, g)
    tables = torch.tensor([[0, 99], [-3, 1]], dtype=torch.int32, device=cuda)
    ctx = torch.tensor([20, 20], dtype=torch.int32, device=cuda)
    ops.paged_attention_int8(torch.zeros(2, 4, 64, dtype=BF, device=cuda), *cache, tables, ctx, scale=1.0)
    with pytest.raises(ops.KernelError, match="bounds"):
        ops.check_errors(cuda)
    ops.kv_dequant_pages_int8(*cache, tables, ctx)
    with pytest.raises(ops.KernelError, match="bounds"):
        ops.check_errors(cuda)
    before = [t.clone() for t in cache]
    x = torch.zeros(1, 2, 64, dtype=BF, device=cuda)
    ops.kv_store_int8(x, x, torch.tensor([4 * 16], device=cuda), *cache)
    with pytest.raises(ops.KernelError, match="bounds"):
        ops.check_errors(cuda)
    layers = [t[None] for t in cache]
    ops.kv_copy_blocks(layers, layers, torch.tensor([7], dtype=torch.int32, device=cuda),
                       torch.tensor([1], dtype=torch.int32, device=cuda))
    with pytest.raises(ops.KernelError, match="bounds"):
        ops.check_errors(cuda)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))


def test_offsets_past_32_bits(cuda):
    """Blocks whose bytes lie behind 2^31 and 2^32 of one cache tensor: store, read and copy them."""
    nb, hkv, d = 270000, 8, 128  # 4.4 GB a tensor
    cache = [torch.empty(nb, hkv, 16, d, dtype=torch.int8, device=cuda) for _ in range(2)]
    cache += [torch.empty(nb, hkv, device=cuda) for _ in range(2)]
    g = torch.Generator().manual_seed(12)
    blocks = [nb - 1, 140000, 3]
    x, y = torch.randn(40, hkv, d, generator=g).to(BF), torch.randn(40, hkv, d, generator=g).to(BF)
    slots = torch.tensor([blocks[t // 16] * 16 + t % 16 for t in range(40)])
    ops.kv_store_int8(x.to(cuda), y.to(cuda), slots.to(cuda), *cache)
    layers = [t[None] for t in cache]
    ops.kv_copy_blocks(layers, layers, blocks, [nb - 5, 5, 139999])
    ops.check_errors(cuda)
    small = [torch.zeros(4, hkv, 16, d, dtype=torch.int8) for _ in range(2)] + [torch.zeros(4, hkv) for _ in range(2)]
    ref.store_int8(x, torch.arange(40), small[0], small[2])
    ref.store_int8(y, torch.arange(40), small[1], small[3])
    for at in (blocks, [nb - 5, 5, 139999]):
        for got, w in zip(cache, small):
            assert torch.equal(got[at].cpu(), w[:3])
        q = torch.randn(1, 32, d, generator=g).to(cuda, BF)
        out = ops.paged_attention_int8(q, *cache, torch.tensor([at], dtype=torch.int32, device=cuda),
                                       torch.tensor([40], dtype=torch.int32, device=cuda), scale=0.1)
        ops.check_errors(cuda)
        want, mass = oracle(q, small, torch.tensor([[0, 1, 2]]), [40], [0, 1], 0.1)
        check(out, want, mass, F16_EPS)


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("hkv", [1, 8])
def test_block_copies(cuda, int8, hkv):
    g = torch.Generator().manual_seed(13)
    L, nb, d = 3, 11, 64
    if int8:
        src = [torch.randint(-128, 128, (L, nb, hkv, 16, d), generator=g, dtype=torch.int8).to(cuda) for _ in range(2)]
        src += [torch.randn(L, nb, hkv, generator=g).to(cuda) for _ in range(2)]
    else:
        src = [torch.randn(L, nb, hkv, 16, d, generator=g).to(cuda, BF) for _ in range(2)]
    want = [t.clone() for t in src]
    ids, to = [4, 9, 4, 0], [1, 2, 3, 10]
    for w in want:
        w[:, to] = w[:, ids]
    ops.kv_copy_blocks(src, src, ids, to)
    ops.check_errors(cuda)
    assert all(torch.equal(a, b) for a, b in zip(src, want))
    dst = [torch.full((L, 6) + tuple(t.shape[2:]), 3, dtype=t.dtype, device=cuda) for t in src]
    i32 = dict(dtype=torch.int32, device=cuda)
    ops.kv_copy_blocks(src, dst, torch.tensor([10, -1, 7], **i32), torch.tensor([5, 1, 0], **i32))
    ops.check_errors(cuda)
    for a, b in zip(src, dst):
        assert torch.equal(b[:, 5], a[:, 10]) and torch.equal(b[:, 0], a[:, 7]) and bool((b[:, 1:5] == 3).all())
    ops.kv_copy_blocks(src, src, [], [])


def test_copy_small_blocks_beside_empty_ones(cuda):
    src = [torch.zeros(2, 5, 0, device=cuda), torch.arange(30., device=cuda).view(2, 5, 3)]
    dst = [torch.zeros_like(t) for t in src]
    ops.kv_copy_blocks(src, dst, [1, 4], [0, 2])
    want = torch.zeros(2, 5, 3, device=cuda)
    want[:, [0, 2]] = src[1][:, [1, 4]]
    assert torch.equal(dst[1], want)
    ops.kv_copy_blocks(src[:1], dst[:1], [1], [0])
    ops.check_errors(cuda)


def test_streams_and_graphs(cuda):
    """A side stream, and two captured graphs of one shape whose replays alternate: every call has its own workspace."""
    g = torch.Generator().manual_seed(14)
    lens = [900, 1700, 64]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 8, 128, g)
    tables = tables.to(cuda)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda)
    qs = [torch.randn(3, 32, 128, generator=g).to(cuda, BF) for _ in range(2)]
    want = [ops.paged_attention_int8(q, *cache, tables, ctx, scale=0.1) for q in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.paged_attention_int8(qs[0], *cache, tables, ctx, scale=0.1)
    side.synchronize()
    assert torch.equal(got, want[0])
    graphs, outs = [], []
    for q in qs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.paged_attention_int8(q, *cache, tables, ctx, scale=0.1))
        graphs.append(gr)
    for _ in range(3):
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    ops.check_errors(cuda)
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    qs[0].copy_(qs[1])
    ctx[0] = 333  # lengths are read at replay
    graphs[0].replay()
    assert torch.equal(outs[0], ops.paged_attention_int8(qs[1], *cache, tables, ctx, scale=0.1))


def test_same_result_every_time(cuda):
    g = torch.Generator().manual_seed(15)
    lens = [5000, 77, 1234]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 8, 128, g)
    q = torch.randn(3, 32, 128, generator=g).to(cuda, BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda)
    first = ops.paged_attention_int8(q, *cache, tables.to(cuda), ctx, scale=0.1)
    for _ in range(20):
        assert torch.equal(first, ops.paged_attention_int8(q, *cache, tables.to(cuda), ctx, scale=0.1))


def test_widest_window(cuda):
    """The largest window is none, for queries in front of the first token too (which see nothing)."""
    g = torch.Generator().manual_seed(21)
    lens, n = [40, 3, 300], [5, 9, 80]
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, 128, g)
    cu = torch.tensor([0, 5, 14, 94], dtype=torch.int32, device=cuda)
    q = torch.randn(94, 4, 128, generator=g).to(cuda, BF)
    args = (tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda))
    for longest in (9, 80):  # read directly, by copies
        c, m = (cu[:3], 14) if longest == 9 else (cu, 94)
        a = [t[:len(c) - 1] for t in args]
        got = [ops.paged_attention_int8(q[:m], *cache, *a, cu_q=c, max_q_len=longest, scale=0.09, window=w)
               for w in (0, 2 ** 31 - 1)]
        assert torch.equal(*got) and not bool(got[1][5:11].any()) and bool(got[1][11:14].any(-1).all())
    ops.check_errors(cuda)


def test_chunk_refusals(cuda):
    """The checks hold on the way through copies too; no head, no group."""
    g = torch.Generator().manual_seed(22)
    cache = make_cache(cuda, 8, 2, 128, g)
    ok = dict(q=torch.zeros(100, 4, 128, dtype=BF, device=cuda), cu_q=torch.tensor([0, 100], dtype=torch.int32,
              device=cuda), tables=torch.arange(8, dtype=torch.int32, device=cuda)[None], max_q_len=100,
              ctx=torch.tensor([120], dtype=torch.int32, device=cuda))

    def attend(q, tables, ctx, **kw):
        return ops.paged_attention_int8(q, *cache, tables, ctx, scale=1.0, **kw)

    attend(**ok)
    bad = [dict(cu_q=ok["cu_q"].cpu()), dict(cu_q=ok["cu_q"].long()), dict(cu_q=torch.zeros(3, dtype=torch.int32,
           device=cuda)), dict(ctx=ok["ctx"].cpu()), dict(sinks=torch.zeros(4)), dict(window=-1), dict(q=ok["q"].cpu()),
           dict(out=torch.zeros(100, 512, dtype=BF, device=cuda)), dict(out=torch.zeros(100, 4, 128, dtype=BF)),
           dict(q=ok["q"].half()), dict(q=ok["q"].transpose(0, 1)), dict(q=ok["q"][:, :0]), dict(q=ok["q"][:, :1]),
           dict(max_q_len=1 << 20), dict(max_q_len=-1), dict(tables=ok["tables"].long())]
    for kw in bad:
        with pytest.raises(RuntimeError, match="b200"):
            attend(**{**ok, **kw})
    ops.check_errors(cuda)


def test_refusals(cuda):
    g = torch.Generator().manual_seed(16)
    cache = make_cache(cuda, 4, 2, 64, g)
    tables = torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    ctx = torch.tensor([20], dtype=torch.int32, device=cuda)
    q = torch.zeros(1, 4, 64, dtype=BF, device=cuda)

    def attend(q=q, cache=cache, tables=tables, ctx=ctx, **kw):
        return ops.paged_attention_int8(q, *cache, tables, ctx, scale=1.0, **kw)

    attend()
    bad = [dict(q=q.float()), dict(q=q[:, :3]), dict(q=torch.zeros(2, 4, 64, dtype=BF, device=cuda)),
           dict(tables=tables.long()), dict(ctx=ctx.repeat(2)), dict(sinks=torch.zeros(3, device=cuda)),
           dict(cache=[cache[0].to(torch.uint8)] + cache[1:]), dict(cache=cache[:3] + [cache[3].double()]),
           dict(cache=cache[:2] + [cache[2][:2], cache[3]]), dict(window=-1), dict(tables=tables.cpu()),
           dict(cu_q=torch.tensor([0, 1, 1], dtype=torch.int32, device=cuda)),
           dict(q=torch.zeros(1, 40, 64, dtype=BF, device=cuda)),
           dict(cache=make_cache(cuda, 2, 2, 32, g), q=torch.zeros(1, 4, 32, dtype=BF, device=cuda))]
    for kw in bad:
        with pytest.raises(RuntimeError, match="b200"):
            attend(**kw)
    x = torch.zeros(1, 2, 64, dtype=BF, device=cuda)
    s = torch.zeros(1, dtype=torch.int64, device=cuda)
    for a in ((x.float(), x, s), (x, x, s.int()), (x, x[:, :1], s), (x, x, s.repeat(2)), (x, x.cpu(), s)):
        with pytest.raises(RuntimeError, match="b200"):
            ops.kv_store_int8(*a, *cache)
    with pytest.raises(RuntimeError, match="b200"):
        ops.kv_copy_blocks([cache[0][None]], [cache[1][None, :, :1]], [0], [1])
    ops.check_errors(cuda)
