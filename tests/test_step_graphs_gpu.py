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
