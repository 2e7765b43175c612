"""The decode-step operators as the engine runs them: a GraniteMoE model with
the CUDA expert layer, attention on the operators, quantised caches, a shared
prefix and sampled tokens, eager and replayed."""
import json

import numpy as np
import pytest
import torch

from gpu_util import require_gpu
from miniep_b200 import Sampler
from miniep_b200.model import (GRANITE_1B_A400M, DeviceModel, Engine, ModelConfig, Shard,
                               random_weights)
from test_gpu_model import _build

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def tiny(golden, **more):
    g = np.load(golden / "model_tiny.npz")
    cfg = ModelConfig.from_dict({**json.loads(str(g["config"])), **more})
    prompts, i = [], 0
    for n in g["prompt_lens"].tolist():
        prompts.append(g["prompts"].tolist()[i:i + n])
        i += n
    return g, cfg, random_weights(cfg, seed=5, dtype=torch.float32), prompts


def close(got, want):
    """fp32 logits by another order of the same sums: the model tests' bound."""
    return (got.cpu() - want.cpu()).abs().max() <= 1e-4 * want.abs().max()


def test_operators_match_the_reference_engine(golden):
    """The reference's prefill and greedy decode, attention on the operators."""
    g, cfg, w, prompts = tiny(golden)
    steps = g["decode_logits"].shape[0]
    comm, placement, _, model = _build(cfg, w, 64, torch.float32)
    eng = Engine(model, reset_rr=placement.reset_rr)
    shard = Shard(prompts, cfg, steps, "cuda", torch.float32, kernels=True)
    eng.prefill(shard)
    assert close(shard.last_prefill_logits, torch.from_numpy(g["prefill_logits"]))
    for t in range(steps):
        eng.decode_step(shard)
        assert close(shard.last_logits, torch.from_numpy(g["decode_logits"][t]))
    assert shard.generated == g["generated"].tolist()
    again = Shard(prompts, cfg, steps, "cuda", torch.float32, kernels=True)
    eng.prefill(again)
    eng.decode_graphed(again, steps)
    assert again.generated == g["generated"].tolist()
    assert close(again.last_logits, torch.from_numpy(g["decode_logits"][steps - 1]))
    comm.check()
    comm.close()


@pytest.mark.parametrize("qk_norm", [False, True])
def test_shared_prefix_is_the_prompt_in_front(golden, qk_norm):
    """prefix + own prompts against the whole prompts, logits and tokens; with
    head norms the plain attention path is the other side too."""
    _, cfg, w, prompts = tiny(golden, qk_norm=qk_norm)
    comm, placement, _, model = _build(cfg, w, 256, torch.float32)
    eng = Engine(model, reset_rr=placement.reset_rr)
    common = torch.randint(1, cfg.vocab_size, (37,), generator=torch.Generator().manual_seed(1)).tolist()
    runs = []
    for kw in (dict(), dict(kernels=True), dict(prefix=eng.build_prefix(common))):
        own = prompts if "prefix" in kw else [common + p for p in prompts]
        shard = Shard(own, cfg, 5, "cuda", torch.float32, **kw)
        eng.prefill(shard)
        first = shard.last_prefill_logits.clone()
        eng.decode_graphed(shard, 5) if kw else [eng.decode_step(shard) for _ in range(5)]
        runs.append((shard.generated, first, shard.last_logits.clone()))
    for other in runs[1:]:
        assert other[0] == runs[0][0]
        assert close(other[1], runs[0][1]) and close(other[2], runs[0][2])
    comm.check()
    comm.close()


@pytest.mark.parametrize("quantized", [False, True])
def test_bf16_steps_replay_and_repeat(quantized):
    """Granite layers in bf16 behind a shared prefix, sampled: eager steps and
    replays draw the same tokens, runs repeat bit for bit, temperature 0 is
    the greedy choice."""
    cfg = ModelConfig.from_dict(dict(GRANITE_1B_A400M, num_hidden_layers=2, vocab_size=4096))
    w = random_weights(cfg, seed=3, dtype=torch.bfloat16)
    gen = torch.Generator().manual_seed(4)
    prompts = [torch.randint(1, 4096, (n,), generator=gen).tolist() for n in (96, 128, 1)]
    comm, placement, _, model = _build(cfg, w, 3 * 128, torch.bfloat16)
    eng = Engine(model, reset_rr=placement.reset_rr)
    prefix = eng.build_prefix(torch.randint(1, 4096, (200,), generator=gen).tolist())

    def run(sampler, graphed):
        shard = Shard(prompts, cfg, 8, "cuda", torch.bfloat16, quantized=quantized, prefix=prefix)
        eng.prefill(shard, sampler=sampler)
        if graphed:
            eng.decode_graphed(shard, 8, sampler=sampler)
        else:
            for _ in range(8):
                eng.decode_step(shard, sampler=sampler)
        assert torch.isfinite(shard.last_logits.float()).all()
        return shard.generated, shard.last_logits.clone()

    filters = dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.01, seed=9)
    first = run(Sampler(**filters), True)
    again = run(Sampler(**filters), True)
    assert first[0] == again[0] and torch.equal(first[1], again[1])
    assert run(Sampler(temperature=0.0), True)[0] == run(None, True)[0]
    eager, greedy = run(Sampler(temperature=0.0), False), run(None, False)
    assert eager[0] == greedy[0] and torch.equal(eager[1], greedy[1])
    other = run(Sampler(**{**filters, "seed": 10}), True)
    assert other[0] != first[0]
    comm.check()
    comm.close()


def test_quantised_cache_holds_what_the_plain_one_does(golden):
    """After a prefill the quantised cache's rows are the plain cache's first
    layer to within e4m3's rounding (2^-4 of a value, 2^-10 of the row's 448th)."""
    _, cfg, w, prompts = tiny(golden)
    comm, placement, _, model = _build(cfg, w, 64, torch.float32)
    eng = Engine(model, reset_rr=placement.reset_rr)
    a = Shard(prompts, cfg, 2, "cuda", torch.float32, kernels=True)
    b = Shard(prompts, cfg, 2, "cuda", torch.float32, quantized=True)
    for s in (a, b):
        eng.prefill(s)
        eng.decode_step(s)
    for x, y in zip(a.cache.read(0, 0, a.T), b.cache.read(0, 0, a.T)):
        top = x.abs().amax(-1, keepdim=True)
        assert ((x - y).abs() <= 2.0 ** -4 * x.abs() * 1.0001 + 2.0 ** -10 * top / 448 * 1.0001).all()
    comm.close()


def test_shard_refuses_positions_past_the_tables(golden):
    _, cfg, w, prompts = tiny(golden)
    comm, placement, _, model = _build(cfg, w, 256, torch.float32)
    prefix = Engine(model, reset_rr=placement.reset_rr).build_prefix(list(range(1, 241)))
    Shard(prompts, cfg, 4, "cuda", torch.float32, prefix=prefix)
    with pytest.raises(ValueError, match="max_position"):
        Shard(prompts, cfg, 5, "cuda", torch.float32, prefix=prefix)
    comm.close()
