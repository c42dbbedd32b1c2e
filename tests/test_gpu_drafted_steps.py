"""The step function with trees of drafted tokens, accepted paths kept, requests that fork, and logits judged on the device: against
the plain model run on every path by itself."""
import os
import re
import subprocess
import sys

import pytest
import torch

import plain_lfm2 as plain
from conftest import TINY
from helpers import ROOT, WEIGHT_STD, assert_close, random_tokens

pytestmark = pytest.mark.gpu
DTYPES = [("float32", torch.float32), ("bfloat16", torch.bfloat16)]


@pytest.fixture(scope="module")
def attention_folders(tmp_path_factory):
    """The tiny models with attention in every layer: no state but keys and values."""
    from celeg_amd.weights import write_random_model
    made = {}

    def get(name, dtype):
        if (name, dtype) not in made:
            cfg, seed = TINY[name]
            cfg = dict(cfg, layer_types=["full_attention"] * cfg["num_hidden_layers"])
            made[name, dtype] = write_random_model(cfg, str(tmp_path_factory.mktemp(f"attention_{name}")), seed=seed, dtype=dtype, std=WEIGHT_STD)
        return made[name, dtype]
    return get


def load(folder, dtype, **options):
    from celeg_amd.engine import load_model
    return load_model(folder, dtype=dtype, **dict(dict(max_requests=4, max_batched_tokens=64), **options))


def feed(lm, slot, tokens, start=0, portion=64):
    from celeg_amd.engine import StepEntry
    for at in range(0, len(tokens), portion):
        part = tokens[at:at + portion]
        assert lm.cache.prepare(slot, start + at, len(part))
        lm.runner.step([StepEntry(slot, start + at, part)])


def way(parents, i):
    out = [i]
    while parents[out[-1]] >= 0:
        out.append(parents[out[-1]])
    return out[::-1]


TREE = [-1, 0, 0, 1, 1, 2, -1, 6, 3, 8, 8]


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
@pytest.mark.parametrize("dtype,stored", DTYPES)
def test_every_path_of_a_tree_is_as_if_it_were_alone(attention_folders, name, dtype, stored):
    from celeg_amd.engine import StepEntry
    folder = attention_folders(name, stored)
    cfg, W = plain.load_model_folder(folder)
    V = cfg["vocab_size"]
    lm = load(folder, dtype)
    assert lm.takes_trees
    # two trees, a single drafted token and a portion of a prompt in one step
    contexts = [random_tokens(V, n, seed=n) for n in (37, 0, 70, 16)]
    trees = [(TREE, random_tokens(V, len(TREE), seed=5)), ([-1, -1, 1], random_tokens(V, 3, seed=6)), ([-1], [3]), ([], random_tokens(V, 4, seed=7))]
    entries = []
    for context, (parents, tokens) in zip(contexts, trees):
        slot = lm.cache.open()
        feed(lm, slot, context)
        assert lm.cache.prepare(slot, len(context), len(tokens))
        entries.append(StepEntry(slot, len(context), tokens, range(len(tokens)), parents))
    got = lm.runner.step(entries)
    assert lm.paths()["attention_trees"] == cfg["num_hidden_layers"]
    row = 0
    for context, (parents, tokens) in zip(contexts, trees):
        parents = parents or [i - 1 for i in range(len(tokens))]
        for i in range(len(tokens)):
            path = [tokens[j] for j in way(parents, i)]
            want = plain.model_logits(cfg, W, context + path)[-1]
            assert_close(got[row + i], want, dtype, f"node {i} behind {len(context)}")
        row += len(tokens)
    lm.close()


@pytest.mark.parametrize("name", ["D", "B"])
@pytest.mark.parametrize("dtype,stored", DTYPES)
def test_the_accepted_path_is_kept_and_goes_on(attention_folders, name, dtype, stored):
    from celeg_amd.engine import StepEntry
    folder = attention_folders(name, stored)
    cfg, W = plain.load_model_folder(folder)
    V = cfg["vocab_size"]
    lm = load(folder, dtype)
    slot = lm.cache.open()
    seq = random_tokens(V, 29, seed=1)
    feed(lm, slot, seq)
    for turn, leaf in enumerate((10, 5, 7, 9)):          # (drafts verified again and again, over page borders)
        tokens = random_tokens(V, len(TREE), seed=50 + turn)
        assert lm.cache.prepare(slot, len(seq), len(TREE))
        lm.runner.step([StepEntry(slot, len(seq), tokens, [leaf], TREE)])
        path = way(TREE, leaf)
        lm.cache.keep(slot, len(seq), [len(seq) + i for i in path])
        lm.cache.check()
        seq = seq + [tokens[i] for i in path]
        assert len(lm.cache.pages_held(slot)[0]) == -(-len(seq) // 16)
    for turn in range(4):                                # decode steps (recorded ones) behind what was kept
        token = random_tokens(V, 1, seed=90 + turn)
        assert lm.cache.prepare(slot, len(seq), 1)
        got = lm.runner.step([StepEntry(slot, len(seq), token, [0])])
        seq = seq + token
        assert_close(got[0], plain.model_logits(cfg, W, seq)[-1], dtype, f"turn {turn}")
    # everything behind the tenth token forgotten, and another way taken from there
    lm.cache.keep(slot, 10)
    other = seq[:10] + random_tokens(V, 9, seed=99)
    assert lm.cache.prepare(slot, 10, 9)
    got = lm.runner.step([StepEntry(slot, 10, other[10:], [8])])
    assert_close(got[0], plain.model_logits(cfg, W, other)[-1], dtype)
    lm.close()


@pytest.mark.parametrize("name", ["A", "D"])
@pytest.mark.parametrize("dtype,stored", DTYPES)
def test_forked_requests_go_their_own_ways(model_folders, name, dtype, stored):
    """(The whole models, with the convolutions' state.)"""
    from celeg_amd.engine import StepEntry
    folder = model_folders(name, stored, WEIGHT_STD)
    cfg, W = plain.load_model_folder(folder)
    V = cfg["vocab_size"]
    lm = load(folder, dtype, n_pages=24)
    first = lm.cache.open()
    seqs = {first: random_tokens(V, 37, seed=3)}
    feed(lm, first, seqs[first])
    free = lm.cache.free_pages()
    for _ in range(2):
        slot = lm.cache.fork(first, 37)
        seqs[slot] = list(seqs[first])
    assert lm.cache.free_pages() == free
    with pytest.raises(ValueError):
        lm.runner.step([StepEntry(first, 37, [1], [0])])          # the last page is shared: prepare first
    for turn in range(6):
        entries = []
        for slot in seqs:
            token = random_tokens(V, 1, seed=100 * slot + turn)
            assert lm.cache.prepare(slot, len(seqs[slot]), 1)
            entries.append(StepEntry(slot, len(seqs[slot]), token, [0]))
            seqs[slot] = seqs[slot] + token
        lm.cache.check()
        got = lm.runner.step(entries)
        for i, e in enumerate(entries):
            assert_close(got[i], plain.model_logits(cfg, W, seqs[e.slot])[-1], dtype, f"slot {e.slot}, turn {turn}")
    # a fork of a fork outlives both
    slot = lm.cache.fork(max(seqs), len(seqs[max(seqs)]))
    seq = list(seqs[max(seqs)])
    for s in seqs:
        lm.cache.close(s)
    more = random_tokens(V, 20, seed=7)
    assert lm.cache.prepare(slot, len(seq), 20)
    got = lm.runner.step([StepEntry(slot, len(seq), more, [19])])
    assert_close(got[0], plain.model_logits(cfg, W, seq + more)[-1], dtype)
    lm.cache.check()
    lm.close()


@pytest.mark.parametrize("name", ["B", "E"])
@pytest.mark.parametrize("dtype,stored", DTYPES)
def test_a_sequence_is_scored(model_folders, name, dtype, stored):
    folder = model_folders(name, stored, WEIGHT_STD)
    cfg, W = plain.load_model_folder(folder)
    V = cfg["vocab_size"]
    lm = load(folder, dtype)
    tokens = random_tokens(V, 100, seed=4)
    logits = plain.model_logits(cfg, W, tokens)[:-1].double()
    want = torch.log_softmax(logits, 1)
    got = lm.score(tokens, top=5, portion=23)
    assert lm.paths()["token_logprobs"] == 5
    at = torch.tensor(tokens[1:])
    # (a log probability is off by as much as two logits are)
    assert_close(got.logprobs[:, 0], want.gather(1, at[:, None])[:, 0], dtype)
    assert_close(got.entropy, -(want.exp() * want).sum(1), dtype)
    assert_close(got.top_logprobs, want.sort(1, descending=True).values[:, :5], dtype)
    if dtype == "float32":
        assert torch.equal(got.top_ids[:, 0].long(), want.argmax(1))
        assert torch.equal(got.ranks[:, 0].long(), (want > want.gather(1, at[:, None])).sum(1))
    assert lm.cache.n_free_slots == 4
    assert lm.score([3]).logprobs.shape == (0, 1) and lm.score([], top=2).top_ids.shape == (0, 2)
    # the device's answers are those of the logits themselves
    from celeg_amd.engine import StepEntry
    slot = lm.cache.open()
    assert lm.cache.prepare(slot, 0, 6)
    judged = lm.runner.logprobs([StepEntry(slot, 0, tokens[:6], [1, 5])], [[0, 1, V - 1], [2, -1, 4]], top=3)
    rows = lm.runner.step([StepEntry(slot, 0, tokens[:6], [1, 5])]).double()
    exact = torch.log_softmax(rows, 1)
    assert (judged.logprobs[0].double() - exact[0, [0, 1, V - 1]]).abs().max() < 1e-5
    assert judged.logprobs[1, 1].isnan() and judged.ranks[1, 1] == -1
    assert torch.equal(judged.top_ids.long(), rows.topk(3).indices)
    assert lm.runner.logprobs([StepEntry(slot, 0, tokens[:6])]).logprobs.shape == (0, 0)
    lm.close()


def test_what_is_refused(model_folders, attention_folders):
    from celeg_amd.engine import StepEntry
    lm = load(model_folders("A", torch.float32, WEIGHT_STD), "float32")
    assert not lm.takes_trees
    slot = lm.cache.open()
    assert lm.cache.prepare(slot, 0, 8)
    with pytest.raises(ValueError, match="trees"):
        lm.runner.step([StepEntry(slot, 0, [1, 2], [0], [-1, 0])])
    with pytest.raises(ValueError, match="state"):
        lm.cache.keep(slot, 0, [0, 2])
    for call in (lambda: lm.runner.logprobs([StepEntry(slot, 0, [1], [0])], [[1] * 9]), lambda: lm.runner.logprobs([StepEntry(slot, 0, [1], [0])], top=129),
                 lambda: lm.runner.logprobs([StepEntry(slot, 0, [1], [0])], [[1], [2]]), lambda: lm.cache.fork(slot, 9), lambda: lm.cache.fork(3, 0)):
        with pytest.raises(ValueError):
            call()
    lm.close()
    lm = load(attention_folders("A", torch.float32), "float32")
    slot = lm.cache.open()
    assert lm.cache.prepare(slot, 0, 8)
    for parents in ([-1], [0, 0], [-1, 1], [-1, -2]):
        with pytest.raises(ValueError):
            lm.runner.step([StepEntry(slot, 0, [1, 2], [0], parents)])
    for start, places in ((-1, [0]), (0, [1, 1]), (0, [2, 1]), (2, [1]), (0, [8]), (0, [20]), (9, [])):
        with pytest.raises(ValueError):
            lm.cache.keep(slot, start, places)
    with pytest.raises(ValueError):
        lm.cache.keep(2, 0)
    assert lm.cache.pages_held(slot) == [[lm.cache.pages_held(slot)[0][0]]]
    lm.close()


def test_keeping_what_two_requests_share(attention_folders):
    """Tokens brought together in one of two requests do not move in the other."""
    from celeg_amd.engine import StepEntry
    folder = attention_folders("D", torch.float32)
    cfg, W = plain.load_model_folder(folder)
    V = cfg["vocab_size"]
    lm = load(folder, "float32")
    a = lm.cache.open()
    seq = random_tokens(V, 20, seed=1)
    feed(lm, a, seq)
    tokens = random_tokens(V, len(TREE), seed=2)
    assert lm.cache.prepare(a, 20, len(TREE))
    lm.runner.step([StepEntry(a, 20, tokens, [], TREE)])
    b = lm.cache.fork(a, 20 + len(TREE))
    kept = {}
    for slot, leaf in ((a, 10), (b, 7)):
        path = way(TREE, leaf)
        lm.cache.keep(slot, 20, [20 + i for i in path])
        kept[slot] = seq + [tokens[i] for i in path]
        lm.cache.check()
    for slot in (a, b):
        assert lm.cache.prepare(slot, len(kept[slot]), 1)
        got = lm.runner.step([StepEntry(slot, len(kept[slot]), [5], [0])])
        assert_close(got[0], plain.model_logits(cfg, W, kept[slot] + [5])[-1], "float32", f"slot {slot}")
    lm.close()


def test_prompt_logprobs_of_the_command_line(model_folders):
    folder = model_folders("D", torch.float32, WEIGHT_STD)
    cfg, W = plain.load_model_folder(folder)
    prompt = random_tokens(cfg["vocab_size"], 12, seed=8)
    proc = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "celeg-run"), "--model", folder, "--dtype", "float32", "--prompt",
                           ",".join(map(str, prompt)), "--max-new-tokens", "2", "--prompt-logprobs", "2"], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stderr
    want = torch.log_softmax(plain.model_logits(cfg, W, prompt).double(), 1)
    lines = re.findall(r"^logprob\[(\d+)\] token=(\d+) logprob=(\S+) rank=(\d+) entropy=(\S+) top=(\S+) (\S+)$", proc.stderr, flags=re.M)
    assert [int(x[0]) for x in lines] == list(range(1, 12)) and [int(x[1]) for x in lines] == prompt[1:]
    for i, line in enumerate(lines):
        assert abs(float(line[2]) - float(want[i, prompt[i + 1]])) < 1e-3       # (printed with four digits)
        assert int(line[5].split(":")[0]) == int(want[i].argmax())
    mean = sum(float(want[i, t]) for i, t in enumerate(prompt[1:])) / 11
    assert abs(float(re.search(r"prompt.mean_logprob=(\S+)", proc.stderr).group(1)) - mean) < 1e-3
