"""What the bf16 copies of int8 pages take: as much as announced, and as long as contexts are, not models."""
import pytest
import torch

from rlx_models_b200 import config as C, ops
from rlx_models_b200.models.decoder import DecoderLM
from rlx_models_b200.runtime.engine import EngineConfig, LLMEngine, SamplingParams
from rlx_models_b200.runtime.speculative import _Seq
from rlx_models_b200.weights.init import random_weights
from test_kv_int8_gpu import BF, make_cache, make_tables

pytestmark = pytest.mark.gpu
MB = 1 << 20


def peak(f):
    """Bytes that the call asks for at its height, beside what is held before it (asked for, not given: the allocator
    hands out blocks of up to a megabyte more)."""
    f()  # (kernels loaded, workspaces made)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    f()
    torch.cuda.synchronize()
    return torch.cuda.memory_stats()["requested_bytes.all.peak"] - before


def test_one_group_of_copies_at_a_time(cuda, monkeypatch):
    g = torch.Generator().manual_seed(3)
    lens = [2048 - 112] * 6  # 121 pages: 128 with those that a box takes, 2 MB for K and V of 2 heads
    tables, nb = make_tables(lens, g)
    cache = make_cache(cuda, nb, 2, 128, g)
    q = torch.randn(6 * 20, 8, 128, generator=g).to(cuda, BF)
    out = torch.empty_like(q)
    args = (q, *cache, tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda))
    kw = dict(cu_q=torch.arange(0, 121, 20, dtype=torch.int32, device=cuda), max_q_len=20, scale=0.1, out=out)
    for limit, groups in ((8 * MB, 4), (4 * MB, 2), (1, 1)):
        monkeypatch.setattr(ops, "INT8_COPY_BYTES", limit)
        taken = peak(lambda: ops.paged_attention_int8(*args, **kw))
        assert groups * 2 * MB <= taken < groups * 2 * MB + MB // 4
    ops.check_errors(cuda)


def tiny():
    return C.tiny(num_hidden_layers=2, hidden_size=256, intermediate_size=256, num_attention_heads=8,
                  num_key_value_heads=2, head_dim=128, vocab_size=512)


def test_an_engine_for_long_contexts(cuda):
    """A prompt of 200 tokens on an engine for 131072: copies of 13 pages, not of 8192 (128 MB)."""
    model = DecoderLM(tiny(), random_weights(tiny(), seed=1), device=cuda)
    eng = LLMEngine(model, EngineConfig(max_num_seqs=4, max_batched_tokens=512, max_model_len=131072, num_blocks=64,
                                        kv_cache_dtype="int8", prefix_caching=False, cuda_graphs=False))
    prompt = torch.randint(0, 512, (200,), generator=torch.Generator().manual_seed(0)).tolist()
    sp = SamplingParams(max_new_tokens=3, ignore_eos=True)
    assert peak(lambda: eng.generate([prompt, prompt[:90]], sp)) < 32 * MB
    ops.check_errors(cuda)


def test_a_speculative_decoder_for_long_contexts(cuda):
    model = DecoderLM(tiny(), random_weights(tiny(), seed=1), device=cuda)
    model.set_kv_cache_dtype("int8")
    s = _Seq(model, 131072)
    assert peak(lambda: s.run(list(range(200)), 0)) < 32 * MB
    ops.check_errors(cuda)
