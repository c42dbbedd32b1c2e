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


@pytest.mark.parametrize("dtype,stored", DTYPES)
@pytest.mark.parametrize("wanted", ["few", "all"])
def test_steps_of_many_rows(tmp_path, dtype, stored, wanted):
    """More rows than the kernels for few of them take, in a model wide enough for the tiled products; with few wanted rows the last
    layer goes on with those alone."""
    from celeg_amd.engine import StepEntry
    from celeg_amd.weights import write_random_model
    cfg, seed = TINY["D"]
    cfg = dict(cfg, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, layer_types=["full_attention"] * cfg["num_hidden_layers"])
    folder = write_random_model(cfg, str(tmp_path), seed=seed, dtype=stored, std=WEIGHT_STD)
    cfg, W = plain.load_model_folder(folder)
    V = cfg["vocab_size"]
    lm = load(folder, dtype, max_batched_tokens=320)
    assert lm.takes_trees
    gen = torch.Generator().manual_seed(8)
    entries, looked = [], []
    for context, n, branches in ((45, 150, True), (0, 83, True), (130, 70, False)):
        slot = lm.cache.open()
        seq = random_tokens(V, context, seed=context)
        if seq:
            feed(lm, slot, seq, portion=320)
        parents = [int(torch.randint(max(-1, i - 6), i, (1,), generator=gen)) for i in range(n)] if branches else []
        tokens = random_tokens(V, n, seed=n)
        assert lm.cache.prepare(slot, context, n)
        nodes = [0, n // 2, n - 1]
        entries.append(StepEntry(slot, context, tokens, nodes if wanted == "few" else range(n), parents))
        for i in nodes:
            looked.append((len(looked) if wanted == "few" else sum(len(e.want) for e in entries[:-1]) + i, seq,
                           [tokens[j] for j in (way(parents, i) if branches else range(i + 1))]))
    got = lm.runner.step(entries)
    assert lm.paths()["attention_trees"] == cfg["num_hidden_layers"]
    for row, seq, path in looked:
        assert_close(got[row], plain.model_logits(cfg, W, seq + path)[-1], dtype, f"row {row}: {len(path)} tokens behind {len(seq)}")
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
    for portion in (0, -3):
        with pytest.raises(ValueError, match="portion"):
            lm.score(tokens, portion=portion)
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


# ---------------------------------------------------------------- layers with and without windows
WINDOWS = (20, None, 7)


def windowed_folder(path, dtype):
    """A model of three attention layers of which two see the last tokens alone, so that their pages are given back early."""
    from celeg_amd.config import LayerSpec, ModelSpec, PartSpec, RunStep, register_architecture, registered_architectures
    from celeg_amd.weights import write_random_model

    def build_spec(cfg, shapes):
        H = cfg["width"]
        norm = lambda name: PartSpec("rmsnorm", {"width": H, "eps": 1e-5}, {"weight": name})
        layers = []
        for i, window in enumerate(WINDOWS):
            p = f"blocks.{i}."
            layers.append(LayerSpec(
                PartSpec("gqa_attention", {"width": H, "heads": 4, "kv_heads": 2, "head_dim": 16, "qk_norm": False, "window": window,
                                           "position": PartSpec("rope", {"theta": 100.0, "head_dim": 16})},
                         {"q_proj": p + "att.q", "k_proj": p + "att.k", "v_proj": p + "att.v", "out_proj": p + "att.o"}),
                norm(p + "n1"), PartSpec("swiglu", {"width": H, "ff": 2 * H}, {"gate": p + "ff.g", "up": p + "ff.u", "down": p + "ff.d"}),
                norm(p + "n2")))
        return ModelSpec("WindowedForCausalLM", cfg["vocab"], H, 256, PartSpec("embedding", {"vocab": cfg["vocab"], "width": H}, {"table": "emb"}),
                         tuple(layers), tuple(RunStep(i) for i in range(len(layers))), norm("final"),
                         PartSpec("tied_head", {"vocab": cfg["vocab"], "width": H}))

    if "WindowedForCausalLM" not in registered_architectures():
        register_architecture("WindowedForCausalLM", build_spec)
    return write_random_model({"architectures": ["WindowedForCausalLM"], "width": 64, "vocab": 91}, path, seed=12, dtype=dtype, std=WEIGHT_STD)


def windowed_logits(W, tokens):
    h = plain.embedding(W["emb"], tokens)
    T = len(tokens)
    for i, window in enumerate(WINDOWS):
        p = f"blocks.{i}."
        n = plain.rmsnorm(h, W[p + "n1"], 1e-5)
        cos, sin = plain.rope_cos_sin(range(T), 100.0, 16)
        q, k, v = (plain.linear(n, W[p + "att." + x]).reshape(T, -1, 16) for x in "qkv")
        o = plain.causal_attention(plain.rope_apply(q, cos, sin), plain.rope_apply(k, cos, sin), v, window=window)
        h = h + plain.linear(o.reshape(T, -1), W[p + "att.o"])
        h = h + plain.swiglu_ffn(plain.rmsnorm(h, W[p + "n2"], 1e-5), W[p + "ff.g"], W[p + "ff.u"], W[p + "ff.d"])
    return plain.linear(plain.rmsnorm(h, W["final"], 1e-5), W["emb"])[-1]


@pytest.mark.parametrize("dtype,stored", DTYPES)
def test_trees_keeps_and_forks_with_windows(tmp_path, dtype, stored):
    from celeg_amd.engine import StepEntry
    folder = windowed_folder(str(tmp_path / "windowed"), stored)
    _, W = plain.load_model_folder(folder)
    lm = load(folder, dtype, page_tokens=4)
    assert lm.takes_trees
    slot = lm.cache.open()
    seqs = {slot: random_tokens(91, 53, seed=1)}
    feed(lm, slot, seqs[slot])
    for turn, leaf in enumerate((10, 7, 9, 5)):
        if turn == 2:
            seqs[lm.cache.fork(slot, len(seqs[slot]))] = list(seqs[slot])
            lm.cache.check()
        entries = []
        for s, seq in seqs.items():
            tokens = random_tokens(91, len(TREE), seed=10 * turn + s)
            assert lm.cache.prepare(s, len(seq), len(TREE))
            entries.append(StepEntry(s, len(seq), tokens, range(len(TREE)), TREE))
        got = lm.runner.step(entries)
        for j, e in enumerate(entries):
            for i in range(len(TREE)):
                assert_close(got[j * len(TREE) + i], windowed_logits(W, seqs[e.slot] + [e.tokens[x] for x in way(TREE, i)]), dtype,
                             f"turn {turn}, slot {e.slot}, node {i}")
            path = way(TREE, leaf)
            lm.cache.keep(e.slot, e.start_pos, [e.start_pos + i for i in path])
            lm.cache.check()
            seqs[e.slot] = seqs[e.slot] + [e.tokens[i] for i in path]
    for s, seq in seqs.items():                         # decoding behind what was kept
        assert lm.cache.prepare(s, len(seq), 1)
        got = lm.runner.step([StepEntry(s, len(seq), [5], [0])])
        assert_close(got[0], windowed_logits(W, seq + [5]), dtype, f"slot {s}")
    # back to before what the windows have given back: refused, as the keys there are gone
    lm.cache.keep(slot, 12)
    assert lm.cache.prepare(slot, 12, 1)
    with pytest.raises(ValueError, match="cover"):
        lm.runner.step([StepEntry(slot, 12, [1], [0])])
    lm.cache.close(slot)
    lm.cache.check()
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
