"""Shared by the host and the GPU test of rolling back int8 pages: models whose
K and V rows are given, so that what a cache holds can be compared bit by bit."""
import torch

from rlx_models_b200.runtime.kv_cache import PagedKVCache
from rlx_models_b200.runtime.speculative import SpeculativeDecoder, _Seq

LAYERS, HKV, D, V = 3, 2, 64, 200
WRONG = 100  # tokens from here on are refused; their rows are 4 times the size


def follows(token, pos):
    return (token * 7 + pos) % 50


class Rows:
    """A decoder with an int8 cache: rows depend on (layer, token, position), the next token on (token, position).
    ``miss(pos)``: answers a wrong token there (a drafter that is refused)."""
    kv_dtype = torch.int8

    def __init__(self, device, miss=lambda pos: False):
        self.device, self.miss = torch.device(device), miss

    def make_kv_cache(self, blocks):
        return PagedKVCache(LAYERS, blocks, HKV, D, device=self.device, dtype=torch.int8)

    def row(self, layer, token, pos):
        g = torch.Generator().manual_seed((layer * 1000 + token) * 1000 + pos)
        return torch.randn(2, HKV, D, generator=g) * (4.0 if token >= WRONG else 1.0)

    def forward(self, fb, kv):
        ids, pos = fb.input_ids.tolist(), fb.positions.tolist()
        for layer in range(LAYERS):
            x = torch.stack([self.row(layer, t, p) for t, p in zip(ids, pos)], 1).bfloat16().to(self.device)
            kv.store_int8(layer, x[0].contiguous(), x[1].contiguous(), fb.slots)
        lg = torch.zeros(len(ids), V, device=self.device)
        for i, (t, p) in enumerate(zip(ids, pos)):
            n = follows(t, p)
            lg[i, n + WRONG if self.miss(p + 1) else n] = 1.0
        return lg


def plain(device, tokens, prompt):
    """The cache after the prompt at once and every further token by itself."""
    s = _Seq(Rows(device), 256)
    s.run(tokens[:prompt], 0)
    for i in range(prompt, len(tokens)):
        s.run([tokens[i]], i)
    return s


def same_cache(a, b, positions):
    blocks = (positions + 15) // 16
    for x, y in zip(a.kv.tensors().values(), b.kv.tensors().values()):
        assert bool((x[:, :blocks] == y[:, :blocks]).all())


def refused_passes_leave_no_trace(device, prompt_len, every):
    """Drafts of four with a refused one among them in every pass: codes and scales are those of plain decoding."""
    prompt = list(range(prompt_len))
    sd = SpeculativeDecoder(Rows(device), Rows(device, lambda pos: pos % every == 0), k=4, max_len=256)
    out = sd.generate(prompt, 40)
    seq = list(prompt)
    while len(seq) < prompt_len + 40:
        seq.append(follows(seq[-1], len(seq) - 1))
    assert prompt + out == seq
    assert 0 < sd.stats.accepted < sd.stats.proposed or every == 1
    same_cache(sd.target, plain(device, seq[:-1], prompt_len), len(seq) - 1)
    return sd
