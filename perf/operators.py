"""The serving cache in 8 bits, its attention, its page copies, and the verification of drafted tokens, as cases that
can be measured.

Four operators, each in the framework's form (``own``) and in elementary torch operations:

* ``attention``: paged attention over int8 pages with one scale per (16-token block, KV head); one query token per
  sequence (decode), a few (verification of drafts) or a chunk of a prompt;
* ``store``: new K / V rows quantised into the pages, then the touched pages as values, as a prompt's attention reads
  them;
* ``copy``: blocks of a cache copied over all layers (the partly filled block of a forked request, a saved prompt);
* ``verify``: drafted tokens accepted or rejected against the target's probabilities from given uniform numbers.

The scale of a block is the smallest power of two ``s`` with ``max |x| <= 127 s``; a code is ``rint(x / s)``.
"""
import math

import torch

own = False

BLOCK = 16
MIN_EXP = -100


def listed():
    """Head counts and sizes: the served dense model (32 query / 8 KV heads of 128), the mixture-of-experts one (64 / 8
    heads of 64, 128-token window, sinks) and the small dense one (16 / 8 heads of 128); vocabulary 151936."""
    return [
        # one short chat turn: latency only
        dict(name="decode one", op="attention", B=1, lo=37, hi=37, hq=32, hkv=8, d=128, n=1, chunk=False, window=0,
             sinks=False, cap=0.0),
        # the serving workload: 64 requests, prompts of 512 to 2048 and up to 256 tokens of output
        dict(name="decode batch", op="attention", B=64, lo=512, hi=2304, hq=32, hkv=8, d=128, n=1, chunk=False,
             window=0, sinks=False, cap=0.0),
        # a sliding-window layer with attention sinks at 128 requests
        dict(name="decode window", op="attention", B=128, lo=1024, hi=1280, hq=64, hkv=8, d=64, n=1, chunk=False,
             window=128, sinks=True, cap=0.0),
        # two very long contexts: the split over the keys carries the parallelism
        dict(name="decode long", op="attention", B=2, lo=131071, hi=131071, hq=16, hkv=8, d=128, n=1, chunk=False,
             window=0, sinks=False, cap=0.0),
        # a verification pass: up to four drafted tokens and the last accepted one
        dict(name="verify pass", op="attention", B=16, lo=800, hi=4000, hq=32, hkv=8, d=128, n=5, chunk=False,
             window=0, sinks=False, cap=0.0),
        # chunks of two prompts over what is cached of them
        dict(name="prompt chunk", op="attention", B=2, lo=4099, hi=8191, hq=32, hkv=8, d=128, n=1024, chunk=True,
             window=0, sinks=False, cap=0.0),
        # the new token of each request of a decode step
        dict(name="store decode", op="store", B=64, n=1, hkv=8, d=128),
        # prompts of a prefill step, of odd lengths
        dict(name="store prompts", op="store", B=7, n=1171, hkv=8, d=128),
        # the partly filled blocks of three forked requests, 8-bit pages and their scales
        dict(name="copy fork", op="copy", pool=64, blocks=3, layers=36, hkv=8, d=128, int8=True, fork=True),
        # a prompt of 4096 tokens taken out of the pool, bf16 pages
        dict(name="copy export", op="copy", pool=288, blocks=256, layers=36, hkv=8, d=128, int8=False, fork=False),
        # one request with four drafts: latency
        dict(name="verify one", op="verify", B=1, k=4, vocab=151936, greedy=0.0, probs=True, spread=3.0),
        # 64 requests with up to four drafts each, an eighth of them greedy
        dict(name="verify batch", op="verify", B=64, k=4, vocab=151936, greedy=0.125, probs=True, spread=3.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "store", "copy", "verify"))
    if op == "attention":
        d = rng.choice((64, 128))
        hkv = rng.choice((1, 2, 4, 8))
        g = rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
        kind = rng.choice(("decode", "decode", "verify", "chunk"))
        if kind == "chunk":
            B, n = rng.choice((1, 2)), _log(rng, 9, 900)
            hi = min(7000, n + _log(rng, 1, 6000))
            g = min(g, 4)
        else:
            B, n = _log(rng, 1, 96), 1 if kind == "decode" else rng.randint(2, 8)
            hi = _log(rng, 8, max(8, min(65536, 140000 // B)))
        return dict(op=op, B=B, lo=max(1, int(hi * rng.uniform(0.05, 1.0))), hi=hi, hq=hkv * g, hkv=hkv, d=d, n=n,
                    chunk=kind == "chunk", window=rng.choice((0, 0, 0, 128, rng.randint(1, 1500))),
                    sinks=rng.random() < 0.3, cap=rng.choice((0.0, 0.0, 0.0, 30.0)))
    if op == "store":
        decode = rng.random() < 0.5
        return dict(op=op, B=_log(rng, 1, 200) if decode else rng.randint(1, 7), n=1 if decode else _log(rng, 2, 1100),
                    hkv=rng.choice((1, 2, 3, 4, 8)), d=rng.choice((64, 128)))
    if op == "copy":
        n = _log(rng, 1, 120)
        return dict(op=op, pool=2 * n + rng.randint(1, 40), blocks=n, layers=rng.choice((1, 5, 24, 28, 36)),
                    hkv=rng.choice((1, 2, 8)), d=rng.choice((64, 128)), int8=rng.random() < 0.5,
                    fork=rng.random() < 0.5)
    return dict(op=op, B=_log(rng, 1, 60), k=rng.randint(1, 4), vocab=_log(rng, 50, 151936),
                greedy=rng.choice((0.0, 0.0, 0.3, 1.0)), probs=rng.random() < 0.7, spread=rng.uniform(0.3, 6.0))


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _new_tokens(case):
    """New tokens of each sequence: the case's number for the first, and down to half of it."""
    return torch.tensor([case["n"] - (37 * b) % (case["n"] // 2 + 1) for b in range(case["B"])])


def _lengths(case, g):
    """Context lengths (the new tokens among them) and new tokens of each sequence."""
    n = _new_tokens(case)
    ctx = torch.randint(case["lo"], case["hi"] + 1, n.shape, generator=g)
    ctx[0] = case["hi"]
    return torch.maximum(ctx, n), n  # every new token is in its own context


def _values(shape, g, dev):
    """Keys or values of each (block, head): rows of about one size per head, a few channels that stand out."""
    x = torch.randn(shape, generator=g, device=dev, dtype=torch.float32)
    head = torch.rand(shape[-3], 1, 1, generator=g, device=dev) * 1.5 + 0.5
    chan = torch.where(torch.rand(shape[-1], generator=g, device=dev) < 0.03, 4.0, 1.0)
    return x.mul_(head).mul_(chan)


def _pow2(amax):
    """Smallest power of two s with amax <= 127 s."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 127.0 / 128.0, e - 7, e - 6).clamp_min(MIN_EXP)
    e = torch.where(amax > 0, e, MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), e)


def _quantised(blocks, hkv, d, g, dev):
    codes = torch.empty(blocks, hkv, BLOCK, d, dtype=torch.int8, device=dev)
    scale = torch.empty(blocks, hkv, dtype=torch.float32, device=dev)
    for at in range(0, blocks, 4096):
        x = _values((min(4096, blocks - at), hkv, BLOCK, d), g, dev)
        s = _pow2(x.abs().amax((2, 3)))
        codes[at:at + 4096] = torch.round(x / s[:, :, None, None]).to(torch.int8)
        scale[at:at + 4096] = s
    return codes, scale


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    gc = torch.Generator()
    gc.manual_seed(seed)
    return dict(case=case, **{"attention": _prepare_attention, "store": _prepare_store, "copy": _prepare_copy,
                              "verify": _prepare_verify}[case["op"]](case, g, gc, dev))


def _prepare_attention(case, g, gc, dev):
    B, hq, hkv, d = case["B"], case["hq"], case["hkv"], case["d"]
    ctx, n = _lengths(case, gc)
    pages = (ctx + BLOCK - 1) // BLOCK
    width, total = int(pages.max()), int(pages.sum())
    order = torch.randperm(total, generator=gc)
    tables = torch.zeros(B, width, dtype=torch.int64)
    held = torch.arange(width)[None, :] < pages[:, None]
    tables[held] = order
    k, ks = _quantised(total, hkv, d, g, dev)
    v, vs = _quantised(total, hkv, d, g, dev)
    T = int(n.sum())
    q = torch.randn(T, hq, d, generator=g, device=dev).to(torch.bfloat16)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)])
    sinks = torch.randn(hq, generator=g, device=dev) if case["sinks"] else None
    return dict(q=q, k=k, v=v, ks=ks, vs=vs, tables=tables.to(dev, torch.int32), ctx=ctx.to(dev, torch.int32),
                cu=cu.to(dev, torch.int32) if case["n"] > 1 else None, max_q=int(n.max()), sinks=sinks,
                scale=1.0 / math.sqrt(d))


def _prepare_store(case, g, gc, dev):
    """Sequences that already hold some tokens get ``n`` more; ``touched`` lists the blocks that change."""
    B, hkv, d = case["B"], case["hkv"], case["d"]
    n = _new_tokens(case)
    first = (11 * torch.arange(B) + 5) % BLOCK  # tokens that the first touched block holds already
    pages = (first + n + BLOCK - 1) // BLOCK
    total = int(pages.sum())
    order = torch.randperm(total + 3, generator=gc)[:total]
    base = torch.cat([torch.zeros(1, dtype=torch.int64), pages.cumsum(0)])
    slots = torch.cat([order[base[b] + (first[b] + torch.arange(int(n[b]))) // BLOCK] * BLOCK
                       + (first[b] + torch.arange(int(n[b]))) % BLOCK for b in range(B)])
    T = int(n.sum())
    k, ks = _quantised(total + 3, hkv, d, g, dev)
    v, vs = _quantised(total + 3, hkv, d, g, dev)
    kn = _values((T, hkv, 1, d), g, dev).view(T, hkv, d).to(torch.bfloat16)
    vn = _values((T, hkv, 1, d), g, dev).view(T, hkv, d).to(torch.bfloat16)
    return dict(kn=kn, vn=vn, slots=slots.to(dev), k=k, v=v, ks=ks, vs=vs,
                touched=order.to(dev, torch.int32).view(-1, 1),
                full=torch.full((total,), BLOCK, dtype=torch.int32, device=dev))


def _prepare_copy(case, g, gc, dev):
    L, pool, hkv, d, n = case["layers"], case["pool"], case["hkv"], case["d"], case["blocks"]
    shape = (L, pool, hkv, BLOCK, d)
    if case["int8"]:
        cache = [torch.randint(-127, 128, shape, generator=g, device=dev, dtype=torch.int8) for _ in range(2)]
        cache += [torch.ldexp(torch.ones(L, pool, hkv, device=dev),
                              torch.randint(-9, -3, (L, pool, hkv), generator=g, device=dev)) for _ in range(2)]
    else:
        cache = [torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2)]
    ids = torch.randperm(pool, generator=gc)
    if case["fork"]:  # into free blocks of the same pool
        dst, to = cache, ids[n:2 * n]
    else:  # into buffers of exactly these blocks
        dst = [torch.empty(L, n, *t.shape[2:], dtype=t.dtype, device=dev) for t in cache]
        to = torch.arange(n)
    return dict(src=cache, dst=dst, ids=ids[:n].to(dev, torch.int32), to=to.to(dev, torch.int32))


def _prepare_verify(case, g, gc, dev):
    """Target logits, and drafts drawn from a drafter that sees them with noise."""
    B, k, V = case["B"], case["k"], case["vocab"]
    n = torch.randint(1, k + 1, (B,), generator=gc)
    n[0] = k
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), (n + 1).cumsum(0)])
    R = int(cu[-1])
    logits = torch.randn(R, V, generator=g, device=dev).mul_(case["spread"])
    temp = torch.rand(B, generator=gc) * 0.9 + 0.5
    temp[torch.rand(B, generator=gc) < case["greedy"]] = 0.0
    rows = torch.cat([torch.arange(int(cu[b]), int(cu[b + 1]) - 1) for b in range(B)]).to(dev)
    noisy = logits[rows] + 0.7 * torch.randn(R - B, V, generator=g, device=dev)
    probs = torch.softmax(noisy, 1)
    if case["probs"]:
        drafts = torch.multinomial(probs, 1, generator=g).view(-1)
    else:
        drafts, probs = noisy.argmax(1), None
    return dict(logits=logits, cu=cu.to(dev, torch.int32), drafts=drafts.to(torch.int32), probs=probs,
                temp=temp.to(dev), u=torch.rand(R, generator=g, device=dev), k=k)


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return {"attention": _own_attention, "store": _own_store, "copy": _own_copy,
                "verify": _own_verify}[state["case"]["op"]](state)
    return {"attention": _plain_attention, "store": _plain_store, "copy": _plain_copy,
            "verify": _plain_verify}[state["case"]["op"]](state)


def _own_attention(s):
    from rlx_models_b200 import ops
    c = s["case"]
    return ops.paged_attention_int8(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["ctx"], cu_q=s["cu"],
                                    max_q_len=s["max_q"], scale=s["scale"], sinks=s["sinks"], window=c["window"],
                                    softcap=c["cap"])


def _own_store(s):
    from rlx_models_b200 import ops
    ops.kv_store_int8(s["kn"], s["vn"], s["slots"], s["k"], s["v"], s["ks"], s["vs"])
    k, v, _ = ops.kv_dequant_pages_int8(s["k"], s["v"], s["ks"], s["vs"], s["touched"], s["full"])
    return dict(k=k, v=v)


def _own_copy(s):
    from rlx_models_b200 import ops
    ops.kv_copy_blocks(s["src"], s["dst"], s["ids"], s["to"])
    return list(s["dst"])


def _own_verify(s):
    from rlx_models_b200 import ops
    tokens, accepted = ops.verify_drafts(s["logits"], s["cu"], s["drafts"], s["probs"], s["temp"], s["u"],
                                         max_drafts=s["k"])
    return dict(tokens=tokens, accepted=accepted)


def _plain_attention(s):
    c = s["case"]
    q, ctx, B = s["q"], s["ctx"].long(), s["ctx"].shape[0]
    T, hq, d = q.shape
    hkv, width = s["k"].shape[1], s["tables"].shape[1]
    at = s["tables"].long().view(-1)

    def rows(codes, scale):
        x = codes[at].float() * scale[at][:, :, None, None]
        return x.view(B, width, hkv, BLOCK, d).transpose(1, 2).reshape(B, hkv, width * BLOCK, d)

    if s["cu"] is None:
        seq, m = torch.arange(B, device=q.device), 1
        idx, new = torch.zeros_like(seq), torch.ones_like(ctx)
    else:
        cu, m = s["cu"].long(), s["max_q"]
        t = torch.arange(T, device=q.device)
        seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
        idx, new = t - cu[seq], cu[1:] - cu[:-1]
    qp = torch.zeros(B, m, hq, d, device=q.device)
    qp[seq, idx] = q.float()
    qp = qp.view(B, m, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, d)
    x = (qp @ rows(s["k"], s["ks"]).transpose(2, 3)).mul_(s["scale"]).view(B, hkv, hq // hkv, m, -1)
    if c["cap"] > 0:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    pos = (ctx - new)[:, None] + torch.arange(m, device=q.device)
    key = torch.arange(width * BLOCK, device=q.device)
    seen = (key <= pos[:, :, None]) & (key < ctx[:, None, None])
    if c["window"] > 0:
        seen &= key > pos[:, :, None] - c["window"]
    x = x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, hkv, hq // hkv, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    o = (p.view(B, hkv, -1, p.shape[-1]) @ rows(s["v"], s["vs"])).view(B, hkv, hq // hkv, m, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, m, hq, d)
    return o[seq, idx].to(q.dtype)


def _plain_store(s):
    def one(new, codes, scale):
        slots = s["slots"]
        block, off = slots // BLOCK, slots % BLOCK
        nb = codes.shape[0]
        x = new.float()
        need = torch.zeros(nb, x.shape[1], device=x.device).index_reduce_(0, block, x.abs().amax(2), "amax")
        hit = torch.zeros(nb, dtype=torch.bool, device=x.device)
        hit[block] = True
        fresh = torch.zeros(nb, device=x.device).index_reduce_(0, block, (off == 0).float(), "amax")
        old = torch.where(fresh[:, None] > 0, 0.0, scale)
        s2 = torch.where(hit[:, None], torch.maximum(old, _pow2(need)), scale)
        kept = torch.round(codes.float() * (old / s2)[:, :, None, None])
        kept[block, :, off] = torch.round(x / s2[block][:, :, None])
        codes.copy_(torch.where(hit[:, None, None, None], kept, codes.float()))
        scale.copy_(s2)
        at = s["touched"].view(-1).long()
        return (codes[at].float() * scale[at][:, :, None, None]).to(torch.bfloat16)

    return dict(k=one(s["kn"], s["k"], s["ks"]), v=one(s["vn"], s["v"], s["vs"]))


def _plain_copy(s):
    ids, to = s["ids"].long(), s["to"].long()
    for a, b in zip(s["src"], s["dst"]):
        b[:, to] = a[:, ids]
    return list(s["dst"])


def _plain_verify(s):
    x, cu, u, k = s["logits"], s["cu"].long(), s["u"].double(), s["k"]
    (R, V), B, dev = x.shape, cu.shape[0] - 1, x.device
    row = torch.arange(R, device=dev)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    n = cu[1:] - cu[:-1] - 1
    top = x.amax(1)
    first = torch.where(x == top[:, None], torch.arange(V, device=dev), V).amin(1)
    temp = s["temp"].double()[seq]
    p = torch.softmax((x.double() - top.double()[:, None]) / torch.where(temp > 0, temp, 1.0)[:, None], 1)
    i = torch.arange(k, device=dev)
    drafted = i < n[:, None]
    at = torch.where(drafted, cu[:-1, None] + i, 0)             # [B, k] rows of the drafts
    dat = torch.where(drafted, at - torch.arange(B, device=dev)[:, None], 0)
    tok = s["drafts"].long()[dat]
    pd = p[at, tok]
    qd = torch.ones_like(pd) if s["probs"] is None else s["probs"].double()[dat, tok]
    greedy = (s["temp"] <= 0)[:, None]
    ok = torch.where(greedy, tok == first[at], u[at] * qd < pd) & drafted
    count = ok.long().cumprod(1).sum(1)
    last = cu[:-1] + count
    w = p[last]
    cut = torch.where(count < n, last - torch.arange(B, device=dev), 0)
    if s["probs"] is None:
        gone = torch.zeros_like(w).scatter_(1, s["drafts"].long()[cut][:, None], 1.0)
    else:
        gone = s["probs"][cut].double()
    w = torch.where((count < n)[:, None], (w - gone).clamp_min(0.0), w)
    c = w.cumsum(1)
    new = (c > (u[cu[1:] - 1] * c[:, -1])[:, None]).long().argmax(1)
    new = torch.where(greedy[:, 0], first[last], new)
    out = torch.full((B, k + 1), -1, dtype=torch.int64, device=dev)
    out[:, :k] = torch.where(i < count[:, None], tok, -1)
    out.scatter_(1, count[:, None], new[:, None])
    return dict(tokens=out.int(), accepted=count.int())


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        ctx, n = _mean_lengths(case)
        pairs, keys = 0.0, 0.0
        for b in range(case["B"]):
            seen = ctx if case["window"] == 0 else min(ctx, case["window"] + n - 1)
            keys += seen
            pairs += n * (seen if n == 1 or case["window"] else ctx - (n - 1) / 2)
        return {"bytes": keys * case["hkv"] * (2 * case["d"] + 8 / BLOCK) + 4 * case["B"] * n * case["hq"] * case["d"],
                "flops": 4.0 * pairs * case["hq"] * case["d"]}
    if case["op"] == "store":
        rows = case["B"] * (case["n"] if case["n"] == 1 else 0.75 * case["n"]) * case["hkv"] * case["d"] * 2
        # bf16 rows read, codes written, codes read again and values written
        return {"bytes": rows * (2 + 1 + 1 + 2), "flops": 4.0 * rows}
    if case["op"] == "copy":
        page = case["hkv"] * (BLOCK * case["d"] * 2 + 8 if case["int8"] else BLOCK * case["d"] * 4)
        return {"bytes": 2.0 * case["layers"] * case["blocks"] * page, "flops": 0.0}
    rows = case["B"] * (1 + (case["k"] + 1) / 2)
    return {"bytes": 4.0 * case["vocab"] * (rows + (case["B"] if case["probs"] else 0)),
            "flops": 5.0 * case["vocab"] * rows}


def _mean_lengths(case):
    n = 1 if case["n"] == 1 else 0.75 * case["n"]
    return max((case["lo"] + case["hi"]) / 2, n), n


# ---------------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "store":
        return _exact_store(s)
    return None  # copies, and whole numbers


def _exact_attention(case, s):
    """Sequence by sequence, head by head."""
    q, out = s["q"].double(), torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group = case["hq"] // case["hkv"]
    ctx = s["ctx"].tolist()
    cu = list(range(case["B"] + 1)) if s["cu"] is None else s["cu"].tolist()
    for b in range(case["B"]):
        at = s["tables"][b, :(ctx[b] + BLOCK - 1) // BLOCK].long()
        new = cu[b + 1] - cu[b]
        pos = torch.arange(ctx[b] - new, ctx[b], device=q.device)[:, None]
        j = torch.arange(ctx[b], device=q.device)[None, :]
        hidden = j > pos
        if case["window"]:
            hidden = hidden | (pos - j >= case["window"])
        for h in range(case["hkv"]):
            key = (s["k"][at, h].double() * s["ks"][at, h].double()[:, None, None]).flatten(0, 1)[:ctx[b]]
            val = (s["v"][at, h].double() * s["vs"][at, h].double()[:, None, None]).flatten(0, 1)[:ctx[b]]
            for r in range(h * group, (h + 1) * group):
                x = torch.einsum("td,jd->tj", q[cu[b]:cu[b + 1], r], key) / math.sqrt(case["d"])
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                x = torch.where(hidden, -math.inf, x)
                if s["sinks"] is not None:
                    x = torch.cat([x, s["sinks"][r].double().expand(new, 1)], 1)
                w = torch.softmax(x, 1)[:, :ctx[b]]
                out[cu[b]:cu[b + 1], r] = torch.einsum("tj,jd->td", w, val)
    return out


def _exact_store(s):
    """The blocks' codes as numbers in 64 bits: amax, exponent by logarithm and correction, rounding to even."""
    def one(new, codes, scale):
        x, slots = new.double(), s["slots"]
        block, off = torch.div(slots, BLOCK, rounding_mode="floor"), slots % BLOCK
        val, sc = codes.double(), scale.double()
        touched = s["touched"].view(-1).long()
        where = torch.full((codes.shape[0],), -1, device=x.device, dtype=torch.long)
        where[touched] = torch.arange(touched.numel(), device=x.device)
        P, H, D = touched.numel(), x.shape[1], x.shape[2]
        rows = torch.zeros(P, BLOCK, H, D, dtype=torch.float64, device=x.device)
        given = torch.zeros(P, BLOCK, dtype=torch.bool, device=x.device)
        rows[where[block], off] = x
        given[where[block], off] = True
        amax = rows.abs().amax((1, 3))
        e = torch.ceil(torch.log2(amax.clamp_min(1e-300) / 127.0))
        e = torch.where(amax > 127.0 * torch.exp2(e), e + 1, e)
        e = torch.where(amax <= 127.0 * torch.exp2(e - 1), e - 1, e).clamp_min(MIN_EXP)
        prev = torch.where(given[:, :1], 0.0, sc[touched])
        now = torch.maximum(torch.exp2(e), prev)
        stay = torch.round(val[touched].permute(0, 2, 1, 3) * (prev / now)[:, None, :, None])
        got = torch.round(rows / now[:, None, :, None])
        got = torch.where(given[:, :, None, None], got, stay) * now[:, None, :, None]
        return got.permute(0, 2, 1, 3).contiguous()

    return dict(k=one(s["kn"], s["k"], s["ks"]), v=one(s["vn"], s["v"], s["vs"]))
