"""The int8 KV cache in use: a served model against the fp32 oracle, chunked
prompts, prompt-cache files, branched requests, and sampled speculative decoding."""
import pytest
import torch

from rlx_models_b200 import config as C
from rlx_models_b200.models.decoder import DecoderLM, ForwardBatch
from rlx_models_b200.models.oracle import DecoderOracle
from rlx_models_b200.registry import build_model
from rlx_models_b200.runtime.engine import EngineConfig, LLMEngine, SamplingParams
from rlx_models_b200.runtime.speculative import SpeculativeDecoder
from rlx_models_b200.weights.init import random_weights

pytestmark = pytest.mark.gpu


def rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def tiny(head_dim):
    return C.tiny(num_hidden_layers=3, hidden_size=512, intermediate_size=1024, num_attention_heads=8,
                  num_key_value_heads=2, head_dim=head_dim, vocab_size=1024)


def engine(model, **kw):
    cfg = dict(max_num_seqs=8, max_batched_tokens=512, max_model_len=512, num_blocks=64, kv_cache_dtype="int8")
    return LLMEngine(model, EngineConfig(**{**cfg, **kw}))


@pytest.mark.parametrize("head_dim", [128, 64])
def test_engine_against_oracle(cuda, head_dim):
    """Codes are off by half a step, at most amax / 127 of a block of 16 rows: about 1.1% of a value's size for normal
    rows (amax 3.5 sigma, steps of amax / 127 to amax / 63, sqrt(12)), beside bf16 activations; three layers of both
    stay below 4% of the logits."""
    cfg = tiny(head_dim)
    w = random_weights(cfg, seed=11, dtype=torch.bfloat16)
    oracle = DecoderOracle(cfg, {k: v.float() for k, v in w.items()})
    model = DecoderLM(cfg, w, device=cuda)
    eng = engine(model, chunk_size=48)
    assert eng.kv.k.dtype == torch.int8
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (100, 1, 37)]
    outs = eng.generate(prompts, SamplingParams(max_new_tokens=12, ignore_eos=True))
    from rlx_models_b200 import ops
    ops.check_errors(cuda)
    for p, o in zip(prompts, outs):
        want, _ = oracle.forward(torch.tensor(p + o.token_ids[:-1]))
        want = want[len(p) - 1:]
        picked = want.gather(1, torch.tensor(o.token_ids)[:, None])[:, 0]
        # a greedy token is the oracle's, or one whose logit is within the two errors of its maximum
        assert bool((picked >= want.amax(1) - 2 * 0.04 * want.norm(dim=1)).all())
    T = 100
    kv = model.make_kv_cache(16)
    fb = ForwardBatch(input_ids=torch.tensor(prompts[0]).int().cuda(), positions=torch.arange(T).int().cuda(),
                      slots=torch.arange(T).cuda(), num_decode=0,
                      pre_block_tables=torch.arange(7, dtype=torch.int32).view(1, -1).cuda(),
                      pre_ctx_lens=torch.tensor([T], dtype=torch.int32).cuda(),
                      pre_cu_q=torch.tensor([0, T], dtype=torch.int32).cuda(), pre_max_q=T)
    lg = model.forward(fb, kv)
    want, _ = oracle.forward(torch.tensor(prompts[0]))
    assert rel(lg.cpu(), want) < 4e-2


def test_bytes_per_block(cuda):
    model = DecoderLM(tiny(128), random_weights(tiny(128), seed=1), device=cuda)
    bf16 = model.kv_bytes_per_block()
    model.set_kv_cache_dtype("int8")
    kv = model.make_kv_cache(5)
    assert sum(t.numel() * t.element_size() for t in kv.tensors().values()) == 5 * model.kv_bytes_per_block()
    assert model.kv_bytes_per_block() < 0.51 * bf16
    with pytest.raises(ValueError, match="int8"):
        model.set_kv_cache_dtype("int4")
    with pytest.raises(NotImplementedError):
        engine(model, kv_retrieval={"topk_blocks": 4})


def test_prompt_cache_roundtrip(cuda, tmp_path):
    model = DecoderLM(tiny(128), random_weights(tiny(128), seed=1), device=cuda)
    prompt = torch.randint(0, 1024, (70,), generator=torch.Generator().manual_seed(0)).tolist()
    sp = SamplingParams(max_new_tokens=6, ignore_eos=True)
    e1 = engine(model)
    first = e1.generate([prompt], sp)[0].token_ids
    path = str(tmp_path / "p.safetensors")
    assert e1.save_prompt_cache(path, prompt) == 64
    e2 = engine(model)
    assert e2.load_prompt_cache(path) == 64
    out = e2.generate([prompt], sp)[0]
    assert out.cached_prompt_tokens == 64
    b1, b2 = e1.sched.prefix_blocks(prompt), e2.sched.prefix_blocks(prompt)
    for t1, t2 in zip(e1.kv.tensors().values(), e2.kv.tensors().values()):
        assert torch.equal(t1[:, b1], t2[:, b2])
    assert out.token_ids == first
    assert engine(model, kv_cache_dtype="bf16").load_prompt_cache(path) == 0


@pytest.mark.parametrize("dtype", ["int8", "bf16", "fp8"])
@pytest.mark.parametrize("asynchronous", [True, False])
@pytest.mark.parametrize("prompt_len", [48, 53])
def test_fork(cuda, dtype, asynchronous, prompt_len):
    """A branch under the same parameters goes on as its parent does (rows of one batch), one under others by
    itself; the copied block is the parent's, and all blocks come back."""
    model = DecoderLM(tiny(128), random_weights(tiny(128), seed=1), device=cuda)
    eng = engine(model, kv_cache_dtype=dtype, async_scheduling=asynchronous, prefix_caching=False)
    free = eng.sched.num_free_blocks()
    prompt = torch.randint(0, 1024, (prompt_len,), generator=torch.Generator().manual_seed(2)).tolist()
    sp = SamplingParams(max_new_tokens=20, ignore_eos=True)
    a = eng.add_request(prompt, sp)
    outs = {}
    for _ in range(5):
        outs.update((o.seq_id, o) for o in eng.step())
    same = eng.fork(a)
    so_far = list(eng.requests[a].tokens)
    assert 0 < len(so_far) < 20
    other = eng.fork(a, SamplingParams(max_new_tokens=9, temperature=1.0, seed=3, ignore_eos=True))
    with pytest.raises(ValueError):
        eng.fork(a + 1000)
    while eng.has_unfinished():
        outs.update((o.seq_id, o) for o in eng.step())
    assert outs[a].token_ids == outs[same].token_ids and len(outs[a].token_ids) == 20
    assert len(outs[other].token_ids) == 9 and outs[other].token_ids[:len(so_far)] == so_far
    assert eng.sched.num_free_blocks() == free
    with pytest.raises(ValueError):
        eng.fork(a)


@pytest.mark.parametrize("mode", ["self", "other", "lookup"])
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_sampled_speculation(cuda, mode, dtype):
    cfg = C.tiny()
    target = build_model(cfg, device=cuda, seed=0)
    draft = {"self": target, "other": build_model(cfg, device=cuda, seed=7), "lookup": None}[mode]
    for m in (target, draft):
        if m is not None:
            m.set_kv_cache_dtype(dtype)
    prompt = torch.randint(0, cfg.vocab_size, (12,), generator=torch.Generator().manual_seed(3)).tolist() * 3
    sd = SpeculativeDecoder(target, draft, k=4, max_len=512)
    greedy = sd.generate(prompt, 24)
    cold = sd.generate(prompt, 24, temperature=1e-4)
    n = 0
    while n < 24 and cold[n] == greedy[n]:
        n += 1
    assert n >= 18  # a draw so cold is the argmax; chunks of other lengths may break a near tie late
    a = sd.generate(prompt, 24, temperature=1.0, seed=5)
    assert a == sd.generate(prompt, 24, temperature=1.0, seed=5)
    assert a != sd.generate(prompt, 24, temperature=1.0, seed=6) and len(a) == 24
    if mode == "self":
        sd = SpeculativeDecoder(target, draft, k=4, max_len=512)
        sd.generate(prompt, 40, temperature=1.0, seed=1)
        assert sd.stats.acceptance > 0.6  # the drafter is the target: refusals are rounding between chunk sizes
