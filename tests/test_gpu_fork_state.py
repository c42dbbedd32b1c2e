"""Models with convolution state: a fork at another length than the one stepped is refused, and one where the state stands goes on rightly."""
import pytest
import torch

import plain_lfm2 as plain
from helpers import WEIGHT_STD, assert_close, random_tokens
from test_gpu_drafted_steps import feed, load

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,stored", [("float32", torch.float32), ("bfloat16", torch.bfloat16)])
def test_forks_of_a_model_with_state(model_folders, dtype, stored):
    from celeg_amd.engine import StepEntry
    folder = model_folders("A", stored, WEIGHT_STD)
    cfg, W = plain.load_model_folder(folder)
    lm = load(folder, dtype, n_pages=24)
    a = lm.cache.open()
    seq = random_tokens(cfg["vocab_size"], 37, seed=3)
    feed(lm, a, seq)
    assert lm.cache.prepare(a, 37, 5)                     # pages ahead of the state
    slots, pages = lm.cache.n_free_slots, lm.cache.free_pages()
    for length in (0, 30, 36, 38, 42):
        with pytest.raises(ValueError, match="state"):
            lm.cache.fork(a, length)
    assert lm.cache.n_free_slots == slots and lm.cache.free_pages() == pages
    b = lm.cache.fork(a, 37)
    for turn in range(4):                                 # (single tokens: recorded steps move the state too)
        if turn == 3:
            with pytest.raises(ValueError, match="behind 40 tokens"):
                lm.cache.fork(b, 37)
        entries = []
        for s in (a, b):
            token = random_tokens(cfg["vocab_size"], 1, seed=10 * turn + s)
            assert lm.cache.prepare(s, 37 + turn, 1)
            entries.append(StepEntry(s, 37 + turn, token, [0]))
        paths = {s: entries[i].tokens for i, s in enumerate((a, b))} if turn == 0 else {s: paths[s] + entries[i].tokens for i, s in enumerate((a, b))}
        got = lm.runner.step(entries)
        for i, s in enumerate((a, b)):
            assert_close(got[i], plain.model_logits(cfg, W, seq + paths[s])[-1], dtype, f"slot {s}, turn {turn}")
    lm.cache.check()
    lm.close()
