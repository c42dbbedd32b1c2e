"""A step of 256 requests of which one has a tree of 256 tokens."""
import pytest
import torch

import plain_lfm2 as plain
from conftest import TINY
from helpers import WEIGHT_STD, assert_close, random_tokens
from test_gpu_drafted_steps import load

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,stored", [("float32", torch.float32), ("bfloat16", torch.bfloat16)])
def test_many_requests_and_one_large_tree(tmp_path, dtype, stored):
    from celeg_amd.engine import StepEntry
    from celeg_amd.weights import write_random_model
    cfg, seed = TINY["D"]
    cfg = dict(cfg, layer_types=["full_attention"] * cfg["num_hidden_layers"])
    folder = write_random_model(cfg, str(tmp_path / "attention"), seed=seed, dtype=stored, std=WEIGHT_STD)
    cfg, W = plain.load_model_folder(folder)
    lm = load(folder, dtype, n_pages=300, max_requests=256, max_batched_tokens=600)
    entries = []
    for i in range(256):
        slot, n = lm.cache.open(), 256 if i == 100 else 1
        assert lm.cache.prepare(slot, 0, n)
        entries.append(StepEntry(slot, 0, random_tokens(cfg["vocab_size"], n, seed=i), [n - 1], [j - 1 if j < 30 else j // 2 for j in range(n)]))
    got = lm.runner.step(entries)
    for i in (0, 99, 100, 101, 254, 255):
        path, at = [], len(entries[i].tokens) - 1
        while at >= 0:
            path.append(entries[i].tokens[at])
            at = entries[i].parents[at]
        assert_close(got[i], plain.model_logits(cfg, W, path[::-1])[-1], dtype, f"entry {i}")
    lm.close()
