"""Prompt-cache files written and read a few blocks at a time, also where some
of the blocks are cached already; what the copies take on the device."""
import pytest
import torch

from rlx_models_b200 import config as C
from rlx_models_b200.models.decoder import DecoderLM
from rlx_models_b200.runtime import prompt_cache
from rlx_models_b200.runtime.engine import EngineConfig, LLMEngine, SamplingParams
from rlx_models_b200.weights.init import random_weights

pytestmark = pytest.mark.gpu


def engine(model, dtype):
    return LLMEngine(model, EngineConfig(max_num_seqs=4, max_batched_tokens=512, max_model_len=512, num_blocks=64,
                                         kv_cache_dtype=dtype))


@pytest.mark.parametrize("dtype", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("blocks", [1, 5, 1000])
def test_roundtrip_in_steps(cuda, tmp_path, monkeypatch, dtype, blocks):
    cfg = C.tiny(num_hidden_layers=3, hidden_size=512, intermediate_size=1024, num_attention_heads=8,
                 num_key_value_heads=2, head_dim=128, vocab_size=1024)
    model = DecoderLM(cfg, random_weights(cfg, seed=1), device=cuda)
    prompt = torch.randint(0, 1024, (200,), generator=torch.Generator().manual_seed(0)).tolist()
    sp = SamplingParams(max_new_tokens=4, ignore_eos=True)
    e1, e2 = engine(model, dtype), engine(model, dtype)
    e1.generate([prompt], sp)
    per_block = sum(t[:, :1].numel() * t.element_size() for t in e1.kv.tensors().values())
    monkeypatch.setattr(prompt_cache, "COPY_BYTES", blocks * per_block + per_block // 2)
    path = str(tmp_path / "p.safetensors")

    def peak(f, *args):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_stats()["requested_bytes.all.current"]
        assert f(*args) == 192
        return torch.cuda.memory_stats()["requested_bytes.all.peak"] - before

    e1.save_prompt_cache(path, prompt)
    e2.generate([prompt[:70] + [3, 1, 4]], sp)  # four of the twelve blocks are there already
    small = 1 << 16
    assert peak(e1.save_prompt_cache, path, prompt) <= 2 * min(blocks, 12) * per_block + small
    assert peak(e2.load_prompt_cache, path) <= 2 * min(blocks, 12) * per_block + small
    b1, b2 = e1.sched.prefix_blocks(prompt), e2.sched.prefix_blocks(prompt)
    assert len(b1) == len(b2) == 12
    for t1, t2 in zip(e1.kv.tensors().values(), e2.kv.tensors().values()):
        x, y = t1[:, b1[4:]].contiguous(), t2[:, b2[4:]].contiguous()
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert e2.generate([prompt], sp)[0].cached_prompt_tokens == 192
