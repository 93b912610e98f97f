"""Prefill attention with two query tiles a CTA (more than 148 tiles) in the
modes of the DiT joint attention (query rows placed through the block table) and
of training (dense rows, the log-sum-exp saved), against 64 bits."""
import math

import pytest
import torch

from rlx_models_b200 import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def plain(q, k, v, scale, causal):
    """One sequence [n, Hq, D] over [L, Hkv, D] in 64 bits: output, sum_j p_j |v_j|, log2-sum-exp2, and per row the
    largest sum_i |q_i k_i| of its keys."""
    G = q.shape[1] // k.shape[1]
    q, k, v = q.double().transpose(0, 1), *(t.double().transpose(0, 1).repeat_interleave(G, 0) for t in (k, v))
    s = q @ k.transpose(1, 2) * scale
    n, L = s.shape[1:]
    if causal:
        s = s.masked_fill(torch.arange(L, device=s.device)[None] > torch.arange(L - n, L, device=s.device)[:, None],
                          -math.inf)
    p = torch.softmax(s, 2)
    size = (q.abs() @ k.abs().transpose(1, 2)).amax(2)
    return ((p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1),
            (torch.logsumexp(s, 2) / math.log(2)).transpose(0, 1), size.transpose(0, 1))


def near(got, want, mass):
    """P is rounded to bf16 (half a step: 2^-8 of each weight), then the output (2^-8 of it); fp32 scores and sums of
    128 products and of a row stay below 2^-13 of the mass sum_j p_j |v_j|."""
    bound = (2.0 ** -8 + 2.0 ** -13) * mass + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -7)
    return bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,L,H", [(2, 1040, 12), (2, 1000, 12), (1, 4608, 24), (3, 129, 30)])
def test_rows_through_the_block_table(cuda, B, L, H, causal):
    """9 tiles of 2 x 12 heads (an odd number, the last with 16 rows), lengths that end inside a page, the size of a
    1024 x 1024 image with its text, and 2 tiles a head of which the second has one row. Output rows in a wider tensor."""
    g = torch.Generator(device=cuda).manual_seed(L)
    pages = (L + 15) // 16
    assert B * ((L + 127) // 128) * H > 148
    nb = B * pages + 3
    q = torch.randn(nb * 16, H, 128, device=cuda, generator=g).to(BF)
    k, v = (torch.randn(nb, H, 16, 128, device=cuda, generator=g).to(BF) for _ in range(2))
    table = torch.randperm(nb, device=cuda, generator=g)[:B * pages].int().view(B, pages)
    free = torch.ones(nb * 16, dtype=torch.bool, device=cuda)
    rows = []
    for b in range(B):
        at = (table[b].long()[:, None] * 16 + torch.arange(16, device=cuda)[None]).reshape(-1)[:L]
        rows.append(at)
        free[at] = False
    wide = torch.full((nb * 16, 256 + H * 128), 7.0, dtype=BF, device=cuda)
    cu = torch.arange(B + 1, dtype=torch.int32, device=cuda) * L
    ctx = torch.full((B,), L, dtype=torch.int32, device=cuda)
    ops.prefill_attention(q, k, v, table, ctx, cu, L, scale=0.09, causal=causal, q_paged=True,
                          out=wide[:, 128:128 + H * 128])
    ops.check_errors(cuda)
    out = wide[:, 128:128 + H * 128].reshape(nb * 16, H, 128)
    for b in range(B):
        kk, vv = (t[table[b].long()].transpose(1, 2).reshape(-1, H, 128)[:L] for t in (k, v))
        for h in range(0, H, 6):  # (six heads at a time: 64-bit scores of all would take gigabytes)
            at = slice(h, h + 6)
            want, mass, _, _ = plain(q[rows[b], at], kk[:, at], vv[:, at], 0.09, causal)
            assert near(out[rows[b], at], want, mass), (b, h)
    assert bool((out[free] == 7.0).all()) and bool((wide[:, :128] == 7.0).all())
    assert bool((wide[:, 128 + H * 128:] == 7.0).all())


@pytest.mark.parametrize("B,S,Hq,Hkv", [(2, 1088, 16, 8), (1, 2048, 32, 4), (3, 704, 12, 12), (9, 64, 80, 20)])
def test_training_rows_and_their_gradients(cuda, B, S, Hq, Hkv):
    from rlx_models_b200.train import functional as TF
    rows_tok = 128 * Hkv // Hq
    assert B * ((S + rows_tok - 1) // rows_tok) * Hkv > 148
    g = torch.Generator(device=cuda).manual_seed(S)
    q, k, v = (torch.randn(B, S, h, 128, device=cuda, generator=g).to(BF).requires_grad_() for h in (Hq, Hkv, Hkv))
    out = torch.empty(B * S, Hq, 128, dtype=BF, device=cuda)
    lse = torch.empty(B * S, Hq, device=cuda)
    tables, lens, cu = TF._attn_meta(B, S, cuda)
    scale = 128 ** -0.5
    ops.ext().attn_train_fwd(q.detach().view(B * S, Hq, 128), k.detach().view(B * S, Hkv, 128),
                             v.detach().view(B * S, Hkv, 128), tables, lens, cu, S, scale, out, lse,
                             ops.scratch(cuda).status)
    ops.check_errors(cuda)
    for b in range(B):
        at = slice(b * S, (b + 1) * S)
        want, mass, lw, size = plain(q[b].detach(), k[b].detach(), v[b].detach(), scale, True)
        assert near(out[at], want, mass), b
        # fp32: a score is off by up to 2^-21 of sum |q k|, a sum of S weights by S 2^-24 and 2^-21 of it, the logarithm
        # by 2^-21 of its size and of 1
        bound = math.log2(math.e) * (2.0 ** -21 * size * scale + S * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -21 * (1 + lw.abs())
        assert bool(((lse[at].double() - lw).abs() <= bound).all()), b
    o = TF.attention(q, k, v, causal=True)
    assert torch.equal(o.view(B * S, Hq, 128), out)
    do = torch.randn(o.shape, device=cuda, generator=g).to(BF)
    o.backward(do)
    ops.check_errors(cuda)
    G = Hq // Hkv
    for b in range(B):
        x, y, z = (t[b].detach().double().transpose(0, 1) for t in (q, k, v))
        d = do[b].double().transpose(0, 1)
        s = x @ y.repeat_interleave(G, 0).transpose(1, 2) * scale
        mask = torch.ones(S, S, dtype=torch.bool, device=cuda).triu(1)
        p = torch.softmax(s.masked_fill(mask, -math.inf), 2)
        dp = d @ z.repeat_interleave(G, 0).transpose(1, 2)
        ds = p * (dp - (p * dp).sum(2, keepdim=True)) * scale
        grads = (ds @ y.repeat_interleave(G, 0), (ds.transpose(1, 2) @ x).view(Hkv, G, S, 128).sum(1),
                 (p.transpose(1, 2) @ d).view(Hkv, G, S, 128).sum(1))
        for t, w in zip((q, k, v), grads):
            # P, dS, the saved output and the gradient are rounded to bf16, 2^-8 of each at most
            err = (t.grad[b].double().transpose(0, 1) - w).norm() / w.norm()
            assert float(err) < 4 * 2.0 ** -8
