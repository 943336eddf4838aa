"""The engine over a cache of 8-bit codes with a scale for each (block, kv head): greedy tokens against the CPU model, prefix caching,
copy-on-write and swapping.  Tolerances are those of the engine's unscaled e5m2 cache, whose codes are off by up to 2^-3 of a value
where e4m3's are by 2^-4 and int8's by 1/254 of a block's largest."""
import random
import types

import pytest
import torch

from test_engine_gpu import _check_greedy

pytestmark = pytest.mark.gpu

KINDS = ["int8", "fp8_e4m3"]
TOL = 8e-2


def engine(kind, **more):
    from splitwise_amd import LLM
    return LLM(more.pop("model", "llama-tiny"), kv_cache_dtype=kind, **{**dict(num_gpu_blocks_override=256, max_num_seqs=12,
                                                                               max_model_len=512, swap_space=0.05), **more})


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("model,eager,pipeline", [("llama-tiny", True, False), ("llama-tiny", False, True), ("opt-tiny", True, False),
                                                  ("opt-tiny", False, False)])
def test_greedy_generation_matches_cpu_model(kind, model, eager, pipeline):
    from splitwise_amd import SamplingParams
    random.seed(0)
    llm = engine(kind, model=model, enforce_eager=eager, pipeline_steps=pipeline)
    vocab = llm.llm_engine.model_config.get_vocab_size()
    prompts = [[random.randrange(vocab) for _ in range(n)] for n in (5, 33, 64, 17, 100, 1, 16, 48, 7, 90, 31)]
    outs = llm.generate(prompt_token_ids=prompts, sampling_params=SamplingParams(temperature=0.0, max_tokens=24))
    assert all(len(o.outputs[0].token_ids) == 24 for o in outs)
    _check_greedy(llm, prompts, outs, tol=TOL)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("eager", [True, False])
def test_prefix_caching(kind, eager, monkeypatch):
    """Prompts that share blocks run their remaining tokens over the cache, codes and scales of other requests' blocks included."""
    from splitwise_amd import SamplingParams, _C
    random.seed(7)
    llm = engine(kind, enforce_eager=eager, enable_prefix_caching=True, num_gpu_blocks_override=96)
    calls = []
    orig = _C.ops.context_attention_scaled
    monkeypatch.setattr(_C.ops, "context_attention_scaled", lambda *a, **k: (calls.append(1), orig(*a, **k)))
    vocab = llm.llm_engine.model_config.get_vocab_size()
    shared = [random.randrange(vocab) for _ in range(150)]
    first = [shared + [random.randrange(vocab) for _ in range(n)] for n in (3, 40)]
    params = SamplingParams(temperature=0.0, max_tokens=12)
    outs = list(llm.generate(prompt_token_ids=first, sampling_params=params))
    second = [shared + [random.randrange(vocab) for _ in range(n)] for n in (1, 17, 64)] + [[random.randrange(vocab) for _ in range(30)],
                                                                                            first[0]]
    before = len(calls)
    outs += list(llm.generate(prompt_token_ids=second, sampling_params=params))
    assert len(calls) - before >= llm.llm_engine.model_config.hf_config["num_hidden_layers"]
    _check_greedy(llm, first + second, outs, tol=TOL)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("blocks", [256, 24])
def test_forks_and_preemption(kind, blocks):
    """Sequences of a request share a prompt's blocks until one writes (a copy, scales too); with 24 blocks groups are swapped out and in."""
    from splitwise_amd import SamplingParams
    random.seed(6)
    llm = engine(kind, num_gpu_blocks_override=blocks, max_model_len=256)
    prompts = [[random.randrange(512) for _ in range(n)] for n in (5, 33, 64, 17, 40)]
    forked = SamplingParams(n=3, best_of=4, temperature=1.0, top_k=1, max_tokens=24, seed=3)
    outs = llm.generate(prompt_token_ids=prompts, sampling_params=forked)
    if blocks < 256:
        assert llm.llm_engine.scheduler.num_preemptions > 0
    assert llm.llm_engine.scheduler.block_manager.get_num_free_gpu_blocks() == blocks
    for prompt, out in zip(prompts, outs):
        assert len(out.outputs) == 3
        for one in out.outputs:
            _check_greedy(llm, [prompt], [types.SimpleNamespace(outputs=[one])], tol=TOL)


@pytest.mark.parametrize("kind", KINDS)
def test_blocks_go_with_their_scales(kind):
    """Copies and swaps, with 2 kv heads: 8 bytes of scales a block."""
    from splitwise_amd.config import CacheConfig
    from splitwise_amd.worker.cache_engine import CacheEngine
    config = CacheConfig(16, 0.5, 0, kind)
    config.num_gpu_blocks, config.num_cpu_blocks = 6, 4
    model = types.SimpleNamespace(dtype=torch.bfloat16, get_head_size=lambda: 64, get_num_layers=lambda p: 3, get_num_kv_heads=lambda p: 2)
    cache = CacheEngine(config, model, types.SimpleNamespace(), torch.device("cuda", 0))
    for k, v in cache.gpu_cache:
        for t in (k, v):
            t.random_(0, 256)
        for s in k.scales:
            s.uniform_()
    before = [(k.clone(), v.clone(), *(s.clone() for s in k.scales)) for k, v in cache.gpu_cache]
    cache.copy({1: [2, 3], 4: [5]})
    torch.cuda.synchronize()
    for (k, v), old in zip(cache.gpu_cache, before):
        for now, was in zip((k, v, *k.scales), old):
            assert torch.equal(now, was[[0, 1, 1, 1, 4, 4]])
    cache.swap_out({1: 3, 4: 0})
    torch.cuda.synchronize()
    cache.swap_in({3: 0, 0: 2})
    torch.cuda.synchronize()
    for (k, v), old in zip(cache.gpu_cache, before):
        for now, was in zip((k, v, *k.scales), old):
            assert torch.equal(now, was[[1, 1, 4, 1, 4, 4]])


def test_copies_of_nothing():
    from splitwise_amd.config import CacheConfig
    from splitwise_amd.worker.cache_engine import CacheEngine
    config = CacheConfig(16, 0.5, 0, "int8")
    config.num_gpu_blocks, config.num_cpu_blocks = 3, 1
    model = types.SimpleNamespace(dtype=torch.bfloat16, get_head_size=lambda: 64, get_num_layers=lambda p: 1, get_num_kv_heads=lambda p: 2)
    cache = CacheEngine(config, model, types.SimpleNamespace(), torch.device("cuda", 0))
    cache.gpu_scales.uniform_()
    before = cache.gpu_scales.clone()
    cache.copy({})
    cache.copy({1: []})
    assert torch.equal(cache.gpu_scales, before)
