"""Speculative-sampling verification against its 64-bit definition: acceptance,
the draw from the residual and behind the last draft, greedy rows, certain
drafts, masked and non-finite logits, ties, and the distribution of its draws."""
import pytest
import torch

from rlx_models_b200 import ops
from rlx_models_b200.ops import reference as ref

pytestmark = pytest.mark.gpu


def make(dev, B, k, V, spread, g, greedy=0.3, probs=True):
    n = torch.randint(0, k + 1, (B,), generator=g)
    n[0] = k
    cu = [0]
    for i in n.tolist():
        cu.append(cu[-1] + i + 1)
    R = cu[-1]
    logits = torch.randn(R, V, generator=g) * spread
    temp = torch.rand(B, generator=g) + 0.3
    temp[torch.rand(B, generator=g) < greedy] = 0.0
    rows = [r for b in range(B) for r in range(cu[b], cu[b + 1] - 1)]
    q = torch.softmax(logits[rows] + 0.5 * torch.randn(len(rows), V, generator=g), 1) if rows else torch.zeros(0, V)
    drafts = torch.multinomial(q, 1, generator=g).view(-1) if probs and rows else (
        logits[rows].argmax(1) if rows else torch.zeros(0))
    return dict(logits=logits, cu=cu, drafts=drafts.int(), q=q if probs else None, temp=temp,
                u=torch.rand(R, generator=g), k=k)


def run(dev, c, k=None):
    out, acc = ops.verify_drafts(c["logits"].to(dev), torch.tensor(c["cu"], dtype=torch.int32, device=dev),
                                 c["drafts"].to(dev), None if c["q"] is None else c["q"].to(dev), c["temp"].to(dev),
                                 c["u"].to(dev), max_drafts=c["k"] if k is None else k)
    return out.tolist(), acc.tolist()


def want(c, k=None):
    return ref.verify_drafts(c["logits"], c["cu"], c["drafts"].tolist(), c["q"], c["temp"].tolist(), c["u"].tolist(),
                             c["k"] if k is None else k)


@pytest.mark.parametrize("V", [1, 2, 31, 512, 513, 4096, 8192, 8193, 32000, 151936])
@pytest.mark.parametrize("probs", [True, False])
def test_against_definition(cuda, V, probs):
    g = torch.Generator().manual_seed(V)
    for B, k in ((1, 4), (9, 3), (3, 9)):
        c = make(cuda, B, k, V, 3.0, g, probs=probs)
        assert run(cuda, c) == want(c)


@pytest.mark.parametrize("spread", [0.0, 0.1, 30.0])
def test_flat_and_peaked(cuda, spread):
    """Equal logits put the borders of the running sum closest together; ties go to the lowest index."""
    g = torch.Generator().manual_seed(3)
    c = make(cuda, 24, 4, 50257, spread, g)
    assert run(cuda, c) == want(c)


@pytest.mark.parametrize("T", [1e-4, 1e-5, 3e-6, 1e-6, 1e-7, 3e-8, 1e-8, 3e-9, 1e-9, 1e-12, 1e-20, 1e-37, 1.4e-45])
def test_cold(cuda, T):
    """Temperatures at which neighbouring fp32 logits are many temperatures apart, next to ties of the largest: random
    logits, logits a few of the last places apart around a power of two, and rows around 0."""
    g = torch.Generator().manual_seed(11)
    c = make(cuda, 9, 3, 9001, 4.0, g, greedy=0.0)
    x, V = c["logits"], 9001
    ulp = 2.0 ** -20  # of fp32 numbers from 8 up
    for r in range(0, x.shape[0], 2):
        x[r] = torch.randint(-9, 4, (V,), generator=g) * ulp + (16.0, -8.0, 0.0, 8.0)[r // 2 % 4]
    for r in range(1, x.shape[0], 4):
        x[r, torch.randint(0, V, (3,), generator=g)] = x[r].max()
    c["temp"] = torch.full_like(c["temp"], T)
    at = [r for b in range(9) for r in range(c["cu"][b], c["cu"][b + 1] - 1)]
    c["drafts"] = x[at].argmax(1).int()
    assert run(cuda, c) == want(c)
    c["q"] = None
    assert run(cuda, c) == want(c)


def test_no_drafts_and_fewer_than_given(cuda):
    g = torch.Generator().manual_seed(4)
    c = make(cuda, 5, 0, 1000, 2.0, g)
    assert run(cuda, c) == want(c)
    c = make(cuda, 5, 4, 1000, 0.5, g)
    assert run(cuda, c, 2) == want(c, 2)  # drafts behind max_drafts are not looked at


def test_masked_and_not_finite(cuda):
    g = torch.Generator().manual_seed(5)
    c = make(cuda, 12, 3, 3000, 2.0, g, greedy=0.4)
    x = c["logits"]
    x[torch.rand(x.shape, generator=g) < 0.6] = -float("inf")
    x[torch.rand(x.shape, generator=g) < 0.01] = float("nan")
    x[::5] = -float("inf")          # rows with nothing allowed
    x[3, 17] = x[3, 40] = float("inf")
    x[7] = torch.finfo(torch.float32).min
    c["q"][::4] = float("nan")
    c["drafts"][1], c["drafts"][2] = -1, 3000
    assert run(cuda, c) == want(c)


def test_identical_distributions_accept(cuda):
    """q = p up to rounding: a refusal can leave no residual; the draw then comes from p."""
    V = 777
    x = torch.linspace(-1, 1, V).repeat(2, 1)
    p = torch.softmax(x[:1].double(), 1)
    c = dict(logits=x, cu=[0, 2], drafts=torch.tensor([5], dtype=torch.int32), q=(p * (1 + 1e-3)).float(),
             temp=torch.ones(1), u=torch.tensor([0.99999994, 0.5]), k=1)
    got = run(cuda, c)
    assert got == want(c) and got[1] == [0]


def test_borders_of_the_uniform(cuda):
    g = torch.Generator().manual_seed(6)
    c = make(cuda, 6, 2, 4097, 1.0, g, greedy=0.0)
    for u in (0.0, 0.99999994, 0.5):
        c["u"] = torch.full_like(c["u"], u)
        assert run(cuda, c) == want(c)


def test_strided_rows_streams_and_graphs(cuda):
    g = torch.Generator().manual_seed(7)
    c = make(cuda, 7, 4, 5001, 2.0, g)
    wide = torch.full((c["logits"].shape[0], 5100), 50.0, device=cuda)
    wide[:, 3:5004] = c["logits"].to(cuda)
    args = (torch.tensor(c["cu"], dtype=torch.int32, device=cuda), c["drafts"].to(cuda), c["q"].to(cuda),
            c["temp"].to(cuda), c["u"].to(cuda))
    w = want(c)
    out, acc = ops.verify_drafts(wide[:, 3:5004], *args, max_drafts=4)
    assert (out.tolist(), acc.tolist()) == w
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, acc = ops.verify_drafts(wide[:, 3:5004], *args, max_drafts=4)
    side.synchronize()
    assert (out.tolist(), acc.tolist()) == w
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, acc = ops.verify_drafts(wide[:, 3:5004], *args, max_drafts=4)
    for _ in range(2):
        gr.replay()
    assert (out.tolist(), acc.tolist()) == w
    ops.check_errors(cuda)


def test_draws_follow_the_target(cuda):
    """Whatever the drafter proposes, the first token is distributed as the target's softmax."""
    g = torch.Generator().manual_seed(8)
    V, B = 8, 16384
    t = torch.randn(V, generator=g)
    q = torch.softmax(torch.randn(V, generator=g), 0)
    drafts = torch.multinomial(q.repeat(B, 1), 1, generator=g).view(-1).int()
    c = dict(logits=t.repeat(2 * B, 1), cu=list(range(0, 2 * B + 1, 2)), drafts=drafts, q=q.repeat(B, 1),
             temp=torch.full((B,), 0.7), u=torch.rand(2 * B, generator=g), k=1)
    out, _ = run(cuda, c)
    freq = torch.bincount(torch.tensor([o[0] for o in out]), minlength=V).double() / B
    p = torch.softmax(t.double() / 0.7, 0)
    assert bool(((freq - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all())  # five standard deviations


def test_refusals(cuda):
    g = torch.Generator().manual_seed(9)
    c = make(cuda, 3, 2, 100, 1.0, g)
    ok = [c["logits"].to(cuda), torch.tensor(c["cu"], dtype=torch.int32, device=cuda), c["drafts"].to(cuda),
          c["q"].to(cuda), c["temp"].to(cuda), c["u"].to(cuda)]
    ops.verify_drafts(*ok, max_drafts=2)
    for i, bad in ((0, ok[0].half()), (0, ok[0].t()), (1, ok[1].long()), (1, ok[1][1:]), (2, ok[2][1:]),
                   (3, ok[3][:, 1:]), (3, ok[3].double()), (4, ok[4].double()), (5, ok[5][1:]), (5, ok[5].cpu())):
        args = list(ok)
        args[i] = bad
        with pytest.raises(RuntimeError, match="b200"):
            ops.verify_drafts(*args, max_drafts=2)
