"""The operators around drafted and forked continuations of requests, measured one call at a time.

Four operators that a program calls between the steps of a model whose keys and values lie in pages:

* ``token_logprobs``: what rows of logits say about given tokens (log probability, rank), their entropy and
  their best alternatives;
* ``tree_attention``: the rows of a tree of drafted tokens over their request's cached context, each seeing the
  context, its ancestors and itself;
* ``move_tokens``: the cached tokens of an accepted (or kept) path brought together, in all layers at once;
* ``copy_pages``: whole pages copied, for a request that goes on in two ways.

Where ``own`` is false the operators are computed from elementary torch operations in 32 bits; where it is true
through ``celeg_amd.ops``.  Sizes: the heads, layers, pages and vocabulary of the models this engine is
benchmarked on (16 heads over 8 of 64, 32 over 8 of 64, 6 attention layers, pages of 16 tokens, 65,536 logits)
and generic ones (heads of 128, other vocabularies).
"""
import math
import random

import torch

own = False

if torch.cuda.is_available():
    DEVICE = "cuda"
else:
    DEVICE = "cpu"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "bfloat16": 2}


def _ops():
    from celeg_amd import ops
    return ops


# ------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # one request that decodes and reports the chosen token and five alternatives: latency alone
        dict(name="logprobs 1x65536 top5", op="logprobs", rows=1, vocab=65536, pad=0, tokens=1, top=5, dtype="float32"),
        # 64 requests that decode together, twenty alternatives each
        dict(name="logprobs 64x65536 top20", op="logprobs", rows=64, vocab=65536, pad=0, tokens=1, top=20, dtype="float32"),
        # a prompt of 2,048 tokens scored (perplexity, ranking of answers)
        dict(name="logprobs 2048x65536 top5", op="logprobs", rows=2048, vocab=65536, pad=0, tokens=1, top=5, dtype="float32"),
        # the rows of several drafted trees, four children looked up in each, an odd vocabulary in a padded buffer
        dict(name="logprobs 333x100003 bf16 top8", op="logprobs", rows=333, vocab=100003, pad=5, tokens=4, top=8, dtype="bfloat16"),
        # one chat with a small tree at a short context: latency alone
        dict(name="tree 1x8 at 700", op="tree", requests=1, nodes=8, nodes_min=8, context=700, context_min=700, heads=16, kv_heads=8,
             dim=64, page=16, layers=6, window=0, dtype="bfloat16"),
        # eight ragged requests with trees of up to 26 nodes
        dict(name="tree 8x26 at 4096", op="tree", requests=8, nodes=26, nodes_min=11, context=4096, context_min=1900, heads=32, kv_heads=8,
             dim=64, page=16, layers=2, window=0, dtype="bfloat16"),
        # sixteen long requests, trees of 64 nodes, heads of 128
        dict(name="tree 16x64 at 16384", op="tree", requests=16, nodes=64, nodes_min=64, context=16384, context_min=12001, heads=32, kv_heads=8,
             dim=128, page=16, layers=1, window=0, dtype="bfloat16"),
        # the 32-bit path, in a sliding window, nodes and contexts odd
        dict(name="tree 3x13 at 1500 window f32", op="tree", requests=3, nodes=13, nodes_min=5, context=1500, context_min=333, heads=16,
             kv_heads=8, dim=64, page=16, layers=2, window=512, dtype="float32"),
        # after a verification: up to five accepted tokens of trees of 32 nodes, 32 requests, six layers, in place
        dict(name="move 32x5 accepted", op="move", requests=32, kept=5, kept_min=1, context=700, layers=6, kv_heads=8, dim=64, page=16,
             spread=0, dtype="bfloat16"),
        # long requests of which a half of the tokens is kept, into pages of a request of their own
        dict(name="move 8x4001 kept", op="move", requests=8, kept=4001, kept_min=3500, context=8192, layers=6, kv_heads=8, dim=64, page=16,
             spread=2, dtype="bfloat16"),
        # a request forked: the page that both go on writing
        dict(name="copy 3 pages", op="copy", pages=3, layers=6, kv_heads=8, dim=64, page=16, dtype="bfloat16"),
        # 64 requests of 1,024 tokens taken over whole
        dict(name="copy 4096 pages", op="copy", pages=4096, layers=6, kv_heads=8, dim=64, page=16, dtype="bfloat16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    op = rng.choice(["logprobs", "logprobs", "tree", "tree", "tree", "move", "copy"])
    if op == "logprobs":
        rows, vocab = _log_int(rng, 1, 2048), _log_int(rng, 1000, 200000)
        rows = max(1, min(rows, 2048 * 65536 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 8, 61]), tokens=rng.randint(1, 8),
                    top=rng.choice([0, 1, 3, 5, 10, 20, 64, 128]), dtype=dtype)
    if op == "tree":
        requests, nodes, context = _log_int(rng, 1, 16), _log_int(rng, 1, 64), _log_int(rng, 16, 16384)
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([32, 64, 64, 96, 128])
        if dtype == "float32":
            requests, nodes, context = min(requests, 4), min(nodes, 32), min(context, 4096)
        return dict(op=op, requests=requests, nodes=nodes, nodes_min=rng.randint(1, nodes), context=context,
                    context_min=rng.randint(0, context), heads=min(kv_heads * group, 32) // kv_heads * kv_heads, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([16, 16, 32]), layers=rng.choice([1, 2]), window=rng.choice([0, 0, 0, _log_int(rng, 1, context)]),
                    dtype=dtype)
    layers, kv_heads, dim = rng.randint(1, 6), rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 96, 128])
    if op == "move":
        spread = rng.choice([0, 2, 3])
        kept = rng.randint(1, 8) if spread == 0 else _log_int(rng, 2, 2000)
        return dict(op=op, requests=_log_int(rng, 1, 32 if spread == 0 else 8), kept=kept, kept_min=rng.randint(1, kept),
                    context=kept * max(spread, 1) + rng.randint(60, 500), layers=layers, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([16, 16, 32]), spread=spread, dtype=dtype)
    return dict(op=op, pages=_log_int(rng, 1, 2048), layers=layers, kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 32]), dtype=dtype)


def _ragged(most, least, n):
    """n lengths from most down to least, the first the longest."""
    return [most - (most - least) * i // max(n - 1, 1) for i in range(n)]


# ------------------------------------------------------------------------------------------------ inputs


def _pages_for(tokens, page):
    return (tokens + page - 1) // page


def _cache(case, lengths, gen, perm_seed, spare=0):
    """Pages of random keys and values, a table whose rows name them in a random order, -1 behind a request's last page."""
    page, dtype = case["page"], TYPES[case["dtype"]]
    counts = [_pages_for(n, page) for n in lengths]
    n_pages, width = sum(counts) + spare, max(counts) + 1
    order = list(range(n_pages))
    random.Random(perm_seed).shuffle(order)
    table, used = [], 0
    for c in counts:
        table.append(order[used:used + c] + [-1] * (width - c))
        used += c
    table.append([n_pages] * width)                    # the row of padded requests: the spare page behind the pool
    shape = (n_pages + 1, case["layers"], case["kv_heads"])
    k = torch.randn(shape + (page, case["dim"]), generator=gen, device=DEVICE, dtype=torch.float32 if DEVICE == "cpu" else dtype)
    v = torch.randn(shape + (case["dim"], page), generator=gen, device=DEVICE, dtype=torch.float32 if DEVICE == "cpu" else dtype)
    return k.to(dtype), v.to(dtype), torch.tensor(table, dtype=torch.int32, device=DEVICE)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed * 7919 + 17)
    state = dict(case=case)
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # a spread of scores with a few tokens far above it, as a trained model's
        wide = torch.randn((rows, vocab + case["pad"]), generator=gen, device=DEVICE) * 2.5
        peaks = torch.randint(0, vocab, (rows, 12), generator=gen, device=DEVICE)
        wide.scatter_add_(1, peaks, torch.rand((rows, 12), generator=gen, device=DEVICE) * 12.0)
        state["logits"] = wide.to(TYPES[case["dtype"]])[:, :vocab]
        tokens = torch.randint(0, vocab, (rows, case["tokens"]), generator=gen, device=DEVICE)
        tokens[:, :1] = peaks[:, :1]
        state["tokens"] = tokens.to(torch.int32)
    elif case["op"] == "tree":
        n = case["requests"]
        contexts, nodes = _ragged(case["context"], case["context_min"], n), _ragged(case["nodes"], case["nodes_min"], n)
        state["k"], state["v"], state["table"] = _cache(case, [c + t for c, t in zip(contexts, nodes)], gen, seed)
        parents = []
        for t in nodes:
            for i in range(t):                         # a few wide levels, as drafts of several tokens at each place give
                parents.append(-1 if i == 0 else rng.randint(max(0, (i - 1) // 4), max(0, (i - 1) // 2)))
        width = case["heads"] * case["dim"]
        state["q"] = torch.randn((sum(nodes), width), generator=gen, device=DEVICE).to(TYPES[case["dtype"]])
        state.update(slots=_ints(list(range(n))), starts=_ints(contexts), offsets=_ints(_offsets(nodes)), parents=_ints(parents),
                     contexts=contexts, nodes=nodes, layer=case["layers"] - 1)
    elif case["op"] == "move":
        n, spread = case["requests"], case["spread"]
        kept = _ragged(case["kept"], case["kept_min"], n)
        if spread == 0:
            # the accepted path of a tree of 32 nodes behind the context, moved up to follow it; the moved nodes
            # lie behind the places they go to, as those of a tree with wide levels do
            lengths, places = [case["context"] + 32] * n, []
            for m in kept:
                places += [case["context"]] + sorted(case["context"] + p for p in rng.sample(range(m, 32), m - 1))
            slots = list(range(n))
            state.update(src=_ints(slots), dst=_ints(slots), starts=_ints([case["context"]] * n))
        else:
            # about one of `spread` tokens kept, into a request of its own
            lengths, places = [case["context"]] * n + [m + 5 for m in kept], []
            for m in kept:
                places += sorted(rng.sample(range(min(case["context"], m * spread)), m))
            state.update(src=_ints(list(range(n))), dst=_ints(list(range(n, 2 * n))), starts=_ints([5] * n))
        state["k"], state["v"], state["table"] = _cache(case, lengths, gen, seed)
        state.update(offsets=_ints(_offsets(kept)), places=_ints(places))
    else:
        n = case["pages"]
        state["k"], state["v"], state["table"] = _cache(case, [2 * n * case["page"]], gen, seed)
        pages = list(range(2 * n))
        rng.shuffle(pages)
        state.update(src=_ints(pages[:n]), dst=_ints(pages[n:]))
    if own and "k" in state:
        state["cache"] = _ops().PagedCache(state["k"], state["v"], state["table"])
    return state


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return _RUN_OWN[op](state)
    return _RUN_PLAIN[op](state)


def _own_logprobs(s):
    r = _ops().token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    return dict(logprobs=r.logprobs, ranks=r.ranks, entropy=r.entropy, top_ids=r.top_ids, top_logprobs=r.top_logprobs)


def _own_tree(s):
    case = s["case"]
    return _ops().tree_attention(s["q"], s["cache"], s["layer"], s["slots"], s["starts"], s["offsets"], s["parents"],
                                 scale=case["dim"] ** -0.5, window=case["window"], max_nodes=case["nodes"],
                                 max_context=case["context"])


def _own_move(s):
    _ops().move_tokens(s["cache"], s["src"], s["dst"], s["offsets"], s["places"], s["starts"])
    return s["k"], s["v"]


def _own_copy(s):
    _ops().copy_pages(s["cache"], s["src"], s["dst"])
    return s["k"], s["v"]


def _plain_logprobs(s):
    x, tokens, top = s["logits"].float(), s["tokens"].long(), s["case"]["top"]
    high = x.amax(1, keepdim=True)
    e = torch.exp(x - high)
    total = e.sum(1, keepdim=True)
    lse = high + torch.log(total)
    at = x.gather(1, tokens)
    entropy = lse[:, 0] - (e * x).sum(1) / total[:, 0]
    index = torch.arange(x.shape[1], device=x.device)
    ranks = torch.stack([((x > at[:, j:j + 1]) | ((x == at[:, j:j + 1]) & (index < tokens[:, j:j + 1]))).sum(1)
                         for j in range(tokens.shape[1])], 1)
    # the best by (logit falling, index rising): the sort is stable
    best, ids = torch.sort(x, dim=1, descending=True, stable=True)
    return dict(logprobs=at - lse, ranks=ranks.to(torch.int32), entropy=entropy, top_ids=ids[:, :top].to(torch.int32),
                top_logprobs=best[:, :top] - lse)


def _visible(parents, first, n, context, window, device):
    """[n, context + n]: which keys a request's nodes see, and the nodes' depths."""
    p = parents[first:first + n].long()
    seen = torch.eye(n, dtype=torch.bool, device=device)
    up = torch.where(p >= 0, p, torch.full_like(p, n))
    for _ in range(max(1, (n - 1).bit_length())):
        # ancestors of the ancestor that is as far away as what is known reaches
        padded = torch.cat([seen, torch.zeros((1, n), dtype=torch.bool, device=device)])
        seen = seen | padded[up]
        up = torch.cat([up, up.new_full((1,), n)])[up]
    depth = seen.sum(1) - 1
    position = torch.cat([torch.arange(context, device=device), context + depth])
    mask = torch.cat([torch.ones((n, context), dtype=torch.bool, device=device), seen], 1)
    if window > 0:
        mask &= position[None, :] > (context + depth)[:, None] - window
    return mask


def _plain_tree(s):
    case, out, first = s["case"], torch.empty_like(s["q"]), 0
    page, dim, heads, kv_heads = case["page"], case["dim"], case["heads"], case["kv_heads"]
    for r, (context, n) in enumerate(zip(s["contexts"], s["nodes"])):
        keys = context + n
        pages = s["table"][r, :_pages_for(keys, page)].long()
        k = s["k"][pages, s["layer"]].float().transpose(0, 1).reshape(kv_heads, -1, dim)[:, :keys]
        v = s["v"][pages, s["layer"]].float().permute(1, 0, 3, 2).reshape(kv_heads, -1, dim)[:, :keys]
        q = s["q"][first:first + n].float().view(n, kv_heads, heads // kv_heads, dim).permute(1, 2, 0, 3).reshape(kv_heads, -1, dim)
        scores = torch.matmul(q, k.transpose(1, 2).contiguous()) * dim ** -0.5
        mask = _visible(s["parents"], first, n, context, case["window"], q.device)
        scores = scores.view(kv_heads, -1, n, keys).masked_fill(~mask, -math.inf)
        scores = torch.exp(scores - scores.amax(-1, keepdim=True))
        weights = (scores / scores.sum(-1, keepdim=True)).view(kv_heads, -1, keys)
        o = torch.matmul(weights, v.contiguous()).view(kv_heads, heads // kv_heads, n, dim)
        out[first:first + n] = o.permute(2, 0, 1, 3).reshape(n, heads * dim).to(out.dtype)
        first += n
    return out


def _plain_move(s):
    offsets, places, page = s["offsets"].long(), s["places"].long(), s["case"]["page"]
    item = torch.arange(places.shape[0], device=places.device)
    request = torch.searchsorted(offsets, item, right=True) - 1
    to = s["starts"].long()[request] + item - offsets[request]
    table = s["table"].long()
    from_page, to_page = table[s["src"].long()[request], places // page], table[s["dst"].long()[request], to // page]
    moved_k, moved_v = s["k"][from_page, :, :, places % page], s["v"][from_page, :, :, :, places % page]
    s["k"][to_page, :, :, to % page] = moved_k
    s["v"][to_page, :, :, :, to % page] = moved_v
    return s["k"], s["v"]


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][dst] = s["k"][src]
    s["v"][dst] = s["v"][src]
    return s["k"], s["v"]


_RUN_OWN = dict(logprobs=_own_logprobs, tree=_own_tree, move=_own_move, copy=_own_copy)
_RUN_PLAIN = dict(logprobs=_plain_logprobs, tree=_plain_tree, move=_plain_move, copy=_plain_copy)


# ------------------------------------------------------------------------------------------------ work


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        # an exponential, its sum and the sum of its products a logit
        return dict(bytes=n * size + case["rows"] * (case["tokens"] * 12 + case["top"] * 8 + 4), flops=4 * n)
    token = case["layers"] * case["kv_heads"] * case["dim"] * 2 * size
    if case["op"] == "tree":
        contexts = _ragged(case["context"], case["context_min"], case["requests"])
        nodes = _ragged(case["nodes"], case["nodes_min"], case["requests"])
        keys, pairs = 0, 0
        for c, t in zip(contexts, nodes):
            reach = min(c, case["window"] - 1) if case["window"] > 0 else c
            keys += reach + t
            pairs += t * (reach + max(1, t.bit_length()))      # (a node's ancestors: a few)
        rows = sum(nodes) * case["heads"] * case["dim"]
        return dict(bytes=keys * case["kv_heads"] * case["dim"] * 2 * size + 2 * rows * size, flops=4 * pairs * case["heads"] * case["dim"])
    if case["op"] == "move":
        return dict(bytes=2 * sum(_ragged(case["kept"], case["kept_min"], case["requests"])) * token, flops=0)
    return dict(bytes=2 * case["pages"] * case["page"] * token, flops=0)


# ------------------------------------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, s)
    if case["op"] == "tree":
        return _exact_tree(case, s)
    # copies: the values themselves, by host indices
    k, v, table, page = s["k"].double(), s["v"].double(), s["table"].tolist(), case["page"]
    if case["op"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            k[b] = k[a]
            v[b] = v[a]
        return k, v
    offsets, places = s["offsets"].tolist(), s["places"].tolist()
    if len(places) > 40000:
        return None
    old_k, old_v = k.clone(), v.clone()
    for r, (a, b, start) in enumerate(zip(s["src"].tolist(), s["dst"].tolist(), s["starts"].tolist())):
        for i, p in enumerate(places[offsets[r]:offsets[r + 1]]):
            old, new = table[a][p // page], table[b][(start + i) // page]
            k[new, :, :, (start + i) % page] = old_k[old, :, :, p % page]
            v[new, :, :, :, (start + i) % page] = old_v[old, :, :, :, p % page]
    return k, v


def _exact_logprobs(case, s):
    parts = []
    for first in range(0, case["rows"], 128):
        x, tokens = s["logits"][first:first + 128].double(), s["tokens"][first:first + 128].long()
        logp = torch.log_softmax(x, 1)
        p = torch.exp(logp)
        best, ids = torch.sort(x, dim=1, descending=True, stable=True)
        place = torch.empty_like(ids).scatter_(1, ids, torch.arange(x.shape[1], device=x.device).expand_as(ids))
        ids = ids[:, :case["top"]]
        parts.append((logp.gather(1, tokens), place.gather(1, tokens).to(torch.int32), -(p * logp).sum(1), ids.to(torch.int32),
                      logp.gather(1, ids)))
    return dict(zip(("logprobs", "ranks", "entropy", "top_ids", "top_logprobs"), (torch.cat(column) for column in zip(*parts))))


def _exact_tree(case, s):
    page, group, window = case["page"], case["heads"] // case["kv_heads"], case["window"]
    q = s["q"].double().view(-1, case["heads"], case["dim"])
    out, parents, first = torch.empty_like(q), s["parents"].tolist(), 0
    for r, (context, n) in enumerate(zip(s["contexts"], s["nodes"])):
        rows = []
        for i in range(n):
            path, at = [], i
            while at >= 0:
                path.append(at)
                at = parents[first + at]
            rows.append(path)
        allowed = torch.zeros((n, context + n), dtype=torch.bool)
        for i, path in enumerate(rows):
            low = 0 if window <= 0 else max(0, context + len(path) - window)      # the node's position less the window, plus one
            allowed[i, low:context] = True
            for up, a in enumerate(path):
                allowed[i, context + a] = window <= 0 or up < window
        allowed = allowed.to(q.device)
        token = torch.arange(context + n, device=q.device)
        where = s["table"][r].long()[token // page]
        for h in range(case["kv_heads"]):
            keys = s["k"][where, s["layer"], h, token % page].double()
            values = s["v"][where, s["layer"], h, :, token % page].double()
            for g in range(h * group, (h + 1) * group):
                score = (q[first:first + n, g] @ keys.T * case["dim"] ** -0.5).masked_fill(~allowed, -math.inf)
                out[first:first + n, g] = torch.softmax(score, 1) @ values
        first += n
    return out.view(-1, case["heads"] * case["dim"])
