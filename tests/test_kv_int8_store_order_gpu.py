"""Batches in which the tokens of one block are not adjacent: one run of them is
stored, the others are left out and reported; everything else as if they were not there."""
import pytest
import torch

from rlx_models_b200 import ops
from rlx_models_b200.ops import reference as ref
from test_kv_int8_gpu import BF, make_cache

pytestmark = pytest.mark.gpu


def rows(n, hkv, d, g):
    return torch.randn(n, hkv, d, generator=g).to(BF), torch.randn(n, hkv, d, generator=g).to(BF)


def stored(cache, x, y, slots, keep):
    """What the 64-bit definition leaves of the tokens in ``keep``."""
    want = [t.cpu().clone() for t in cache]
    for i, r in ((0, x), (1, y)):
        ref.store_int8(r[keep], slots[keep], want[i], want[2 + i])
    return want


def same(cache, want):
    return all(torch.equal(a.cpu(), b) for a, b in zip(cache, want))


@pytest.mark.parametrize("hkv,d", [(8, 128), (1, 64)])
@pytest.mark.parametrize("slots,left_out", [
    ([32, 48, 33], [2]),                                # another block between them
    ([32, -1, 33], [2]),                                # a skipped row between them
    ([35, 36, -3, 16, 17, 37, 38, 0], [5, 6]),
    ([48, 32, 49, 33, 50], [2, 3, 4]),
])
def test_the_first_run_is_stored(cuda, slots, left_out, hkv, d):
    g = torch.Generator().manual_seed(1)
    cache = make_cache(cuda, 5, hkv, d, g)
    x, y = rows(len(slots), hkv, d, g)
    slots = torch.tensor(slots)
    want = stored(cache, x, y, slots, [i for i in range(len(slots)) if i not in left_out])
    ops.kv_store_int8(x.to(cuda), y.to(cuda), slots.to(cuda), *cache)
    with pytest.raises(ops.KernelError, match="adjacent"):
        ops.check_errors(cuda)
    assert same(cache, want)


def test_the_last_token_of_the_longest_scan(cuda):
    g = torch.Generator().manual_seed(2)
    for T in (255, 256):
        cache = make_cache(cuda, 300, 2, 64, g)
        x, y = rows(T, 2, 64, g)
        slots = torch.arange(T) * 16
        slots[T - 1] = 5  # its block was the first token's
        want = stored(cache, x, y, slots, list(range(T - 1)))
        ops.kv_store_int8(x.to(cuda), y.to(cuda), slots.to(cuda), *cache)
        with pytest.raises(ops.KernelError, match="adjacent"):
            ops.check_errors(cuda)
        assert same(cache, want)


@pytest.mark.parametrize("T", [257, 900, 1025, 5000])
def test_one_of_the_runs_is_stored(cuda, T):
    g = torch.Generator().manual_seed(T)
    cache = make_cache(cuda, T // 16 + 2, 2, 128, g)
    x, y = rows(T, 2, 128, g)
    slots = torch.arange(T)
    apart = T - 7
    slots[apart] = 20  # in the second block, tokens 16 .. 31
    slots[apart + 1:] = -1  # (the rows behind would be parted from their own block's)
    first = stored(cache, x, y, slots, [i for i in range(T) if i != apart])
    second = stored(cache, x, y, slots, [i for i in range(T) if not 16 <= i < 32])
    ops.kv_store_int8(x.to(cuda), y.to(cuda), slots.to(cuda), *cache)
    with pytest.raises(ops.KernelError, match="adjacent"):
        ops.check_errors(cuda)
    for i in range(4):  # K and V, codes and scales of either run
        assert torch.equal(cache[i].cpu(), first[i]) or torch.equal(cache[i].cpu(), second[i])
    assert same(cache, first) or same(cache, second)


@pytest.mark.parametrize("T", [1, 64, 256, 257, 1024, 1025, 3000])
def test_batches_in_order_report_nothing(cuda, T):
    """Every token in a block of its own, in any order of blocks, and runs of all lengths."""
    g = torch.Generator().manual_seed(T)
    for kind in range(2):
        cache = make_cache(cuda, T + 1, 1, 64, g)
        x, y = rows(T, 1, 64, g)
        if kind == 0:
            slots = torch.randperm(T + 1, generator=g)[:T] * 16 + torch.randint(0, 16, (T,), generator=g)
        else:
            slots = torch.arange(T) + 16 * torch.div(torch.arange(T), 50, rounding_mode="floor")
            slots = slots[slots < (T + 1) * 16]
            x, y = x[:len(slots)], y[:len(slots)]
        want = stored(cache, x, y, slots, list(range(len(slots))))
        ops.kv_store_int8(x.to(cuda), y.to(cuda), slots.to(cuda), *cache)
        ops.check_errors(cuda)
        assert same(cache, want)
