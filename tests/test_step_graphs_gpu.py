"""Middle portions of prompts, which want no logits, from captured graphs: what they leave behind is what eager steps leave."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import test_vopepel_gpu as vopepel
from conftest import TINY_CONFIGS
from test_engine_gpu import engine_for
from test_vopepel_gpu import models   # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def portions(engine, tokens, size=32):
    """One request's tokens in portions without logits, then one token with: its logits."""
    from pylon_b200.engine.step import StepEntry

    request = engine.open("a", len(tokens) + 1)
    for first in range(0, len(tokens), size):
        engine.step([StepEntry(request, tokens[first : first + size])])
    return request, engine.step([StepEntry(request, [3], (0,))]).float()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bits", [4, 16])
def test_every_vote_counts_once(bits, dtype, tiny_folders):
    name = "tinyC"
    fields = TINY_CONFIGS[name]
    tokens = np.random.default_rng(3).integers(0, fields["vocab_size"], size=6 * 32).tolist()
    logits = []
    for graphs in (False, True):
        engine = engine_for(tiny_folders[name], name, dtype, cache_bits=bits, cache_keep=250, cuda_graphs=graphs)
        request, got = portions(engine, tokens)
        logits.append(got)
        assert not graphs or engine.step_function.graphs.replays["padded"] >= 4
        group = engine.cache.groups[0]
        page = torch.tensor(request.tables[0], device=engine.device)
        slots = torch.arange(len(tokens) + 1, device=engine.device)
        mass = group.mass[:, page[slots // engine.cache.page_size], :, slots % engine.cache.page_size].double()
        # every token's weights sum to one: 193 votes of the query heads of a KV head in every layer (a weight and its sum off by 1e-5 at most)
        votes = (len(tokens) + 1) * fields["num_attention_heads"] // fields["num_key_value_heads"]
        assert ((mass.sum(0) - votes).abs() <= 1e-4 * votes).all(), (graphs, mass.sum(0), votes)
    torch.testing.assert_close(logits[0], logits[1], rtol=0, atol=(1e-3 if dtype == "float32" else 0.25) * float(logits[0].std()))   # (the padded step's kernels split its sums otherwise)


def test_states_are_advanced_once(models):   # noqa: F811
    folder, config, weights = models["one_stream"]
    tokens = list(vopepel.make_requests(config, (160,), seed=23).values())[0]
    logits = []
    for graphs in (False, True):
        engine = vopepel.engine_for(folder, "float32", 64, 256, cuda_graphs=graphs)
        logits.append(portions(engine, list(tokens))[1])
        assert not graphs or engine.step_function.graphs.replays["padded"] >= 3
    torch.testing.assert_close(logits[0], logits[1], rtol=0, atol=1e-3 * float(logits[0].std()))


@pytest.mark.parametrize("seed", [0, 1])
@pytest.mark.parametrize("bits, keep", [(4, None), (4, 48), (16, 48)])
def test_prompts_in_many_portions_give_the_tokens_of_eager_steps(bits, keep, seed, tiny_folders):
    """In float32, prompts of up to 200 tokens in portions of 32 beside decoded tokens of other requests: what is evicted, and so every token, is the same."""
    from pylon_b200.sampling import SamplingParams

    name, rng = "tinyC", np.random.default_rng(seed)
    prompts = [rng.integers(0, TINY_CONFIGS[name]["vocab_size"], size=n).tolist() for n in rng.integers(1, 200, size=7)]
    outcomes = []
    for options in (dict(run_ahead=False), dict(cuda_graphs=True, run_ahead=False), dict(cuda_graphs=True)):
        engine = engine_for(tiny_folders[name], name, "float32", cache_bits=bits, cache_keep=keep, prefill_chunk_size=32, max_batch_size=3, **options)
        outcomes.append([result.output_ids for result in engine.generate(prompts, SamplingParams(max_new_tokens=30, temperature=0.0, ignore_eos=True))])
        assert not options.get("cuda_graphs") or engine.step_function.graphs.replays["padded"] > 3
    assert outcomes[0] == outcomes[1] == outcomes[2]
