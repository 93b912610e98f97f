"""Decoding on the int8 cache token by token: logits and picked tokens against
the fp32 oracle by the error of one logit, and branches of a request."""
import math

import pytest
import torch

from rlx_models_b200 import config as C, ops
from rlx_models_b200.models.decoder import DecoderLM, ForwardBatch
from rlx_models_b200.models.oracle import DecoderOracle
from rlx_models_b200.runtime.engine import EngineConfig, LLMEngine, SamplingParams
from rlx_models_b200.weights.init import random_weights

pytestmark = pytest.mark.gpu

# Codes are off by half a step, about 1.1% of a value's size for normal rows (steps of amax / 127 to amax / 63 with amax
# 3.5 sigma, over sqrt(12)), beside bf16 activations; three layers of both stay below 4% of the logits' norm, so the
# error of one logit has a standard deviation of 4% of theirs, that of a difference sqrt(2) of it.
REL = 0.04


def tiny(head_dim):
    return C.tiny(num_hidden_layers=3, hidden_size=512, intermediate_size=1024, num_attention_heads=8,
                  num_key_value_heads=2, head_dim=head_dim, vocab_size=1024)


def build(cuda, head_dim, seed):
    cfg = tiny(head_dim)
    w = random_weights(cfg, seed=seed, dtype=torch.bfloat16)
    return DecoderLM(cfg, w, device=cuda), DecoderOracle(cfg, {k: v.float() for k, v in w.items()})


def engine(model, **kw):
    cfg = dict(max_num_seqs=8, max_batched_tokens=512, max_model_len=512, num_blocks=64, kv_cache_dtype="int8")
    return LLMEngine(model, EngineConfig(**{**cfg, **kw}))


def near_greedy(oracle, prompt, tokens):
    """Every token is the oracle's, or its logit is within six standard deviations of a difference of the largest."""
    want, _ = oracle.forward(torch.tensor(prompt + tokens[:-1]))
    want = want[len(prompt) - 1:].double()
    picked = want.gather(1, torch.tensor(tokens)[:, None])[:, 0]
    slack = 6 * math.sqrt(2) * REL * want.std(dim=1)
    return bool((picked >= want.amax(1) - slack).all())


@pytest.mark.parametrize("head_dim", [128, 64])
def test_logits_of_single_tokens(cuda, head_dim):
    model, oracle = build(cuda, head_dim, 11)
    model.set_kv_cache_dtype("int8")
    kv = model.make_kv_cache(16)
    seq = torch.randint(0, 1024, (150,), generator=torch.Generator().manual_seed(1)).tolist()
    table = torch.arange(16, dtype=torch.int32, device=cuda).view(1, -1)
    n = 100
    model.forward(ForwardBatch(input_ids=torch.tensor(seq[:n]).int().cuda(), positions=torch.arange(n).int().cuda(),
                               slots=torch.arange(n).cuda(), num_decode=0, pre_block_tables=table,
                               pre_ctx_lens=torch.tensor([n], dtype=torch.int32, device=cuda),
                               pre_cu_q=torch.tensor([0, n], dtype=torch.int32, device=cuda), pre_max_q=n), kv)
    want, _ = oracle.forward(torch.tensor(seq))
    for i in range(n, len(seq)):  # through three block ends
        one = lambda x, t: torch.tensor([x], dtype=t, device=cuda)
        lg = model.forward(ForwardBatch(input_ids=one(seq[i], torch.int32), positions=one(i, torch.int32),
                                        slots=one(i, torch.int64), num_decode=1, dec_block_tables=table,
                                        dec_ctx_lens=one(i + 1, torch.int32)), kv)
        assert float((lg[0].cpu().float() - want[i]).norm() / want[i].norm()) < REL
    ops.check_errors(cuda)


@pytest.mark.parametrize("head_dim", [128, 64])
def test_picked_tokens(cuda, head_dim):
    model, oracle = build(cuda, head_dim, 11)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, 1024, (n,), generator=g).tolist() for n in (100, 1, 37)]
    outs = engine(model, chunk_size=48).generate(prompts, SamplingParams(max_new_tokens=40, ignore_eos=True))
    ops.check_errors(cuda)
    for p, o in zip(prompts, outs):
        assert near_greedy(oracle, p, o.token_ids)


@pytest.mark.parametrize("asynchronous", [True, False])
@pytest.mark.parametrize("prompt_len", [48, 53])
def test_branches(cuda, asynchronous, prompt_len):
    """The copied block is the parent's bit for bit, parent and branch share the tokens so far, and each goes on as a
    greedy request does (not necessarily with the same bits: rows of a batch may differ in the last ones)."""
    model, oracle = build(cuda, 128, 1)
    eng = engine(model, async_scheduling=asynchronous, prefix_caching=False)
    prompt = torch.randint(0, 1024, (prompt_len,), generator=torch.Generator().manual_seed(2)).tolist()
    a = eng.add_request(prompt, SamplingParams(max_new_tokens=20, ignore_eos=True))
    for _ in range(5):
        eng.step()
    copied = []
    copy = eng.kv.copy_blocks
    eng.kv.copy_blocks = lambda src, dst: (copied.append((src, dst)), copy(src, dst))
    b = eng.fork(a)
    so_far = list(eng.requests[a].tokens)
    (src, dst), = copied
    for t in eng.kv.tensors().values():
        assert bool((t[:, src] == t[:, dst]).all()) and bool(t[:, dst].any())
    outs = {}
    while eng.has_unfinished():
        outs.update((o.seq_id, o) for o in eng.step())
    ops.check_errors(cuda)
    for sid in (a, b):
        tokens = outs[sid].token_ids
        assert tokens[:len(so_far)] == so_far and len(tokens) == 20
        assert near_greedy(oracle, prompt, tokens)
