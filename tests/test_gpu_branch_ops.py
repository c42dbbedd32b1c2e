"""``celeg_amd.ops`` on the GPU against 64-bit results: sizes, types, masks and lists where the kernels can go wrong."""
import math
import random

import pytest
import torch

from celeg_amd import ops

import plain_branch as plain

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


# ------------------------------------------------------------------------------------------------ log probabilities


def check_logprobs(logits, tokens, top):
    got = ops.token_logprobs(logits, tokens, top=top)
    want = plain.token_logprobs(logits, tokens, top)
    vocab = logits.shape[1]
    finite = logits.float().cpu()
    size = finite[finite.isfinite()].abs().max().item() if finite.isfinite().any() else 0.0
    # a logit less the largest is rounded once, its exponential to a few steps and by the argument's error; a thread adds up to
    # vocab / 256 of them one after the other (at most 1,024 here), the threads' sums are joined in a few more
    chain = min(vocab / 256, 1024) + 64
    near = 2.0 ** -24 * (8 * size + chain + 4 * math.log(vocab + 1))
    for name, g, w in zip(got._fields, got, want):
        if g is None:
            assert w is None
            continue
        g = g.cpu()
        assert g.shape == w.shape, name
        if g.dtype == torch.int32:
            assert torch.equal(g.long(), w), name
            continue
        assert torch.equal(g.isnan(), w.isnan()), name
        ok = ~w.isnan()
        infinite = ok & w.isinf()
        assert torch.equal(g[infinite].double(), w[infinite]), name
        ok &= ~w.isinf()
        # (the entropy's terms are sums of e d: the same relative errors of numbers up to the logarithm of the vocabulary)
        tolerance = near * (4 + math.log(vocab + 1)) if name == "entropy" else near + 2.0 ** -22 * w[ok].abs()
        assert ((g[ok].double() - w[ok]).abs() <= tolerance).all(), (name, (g[ok].double() - w[ok]).abs().max())
    return got


def rows_of(kind, rows, vocab, gen):
    x = torch.randn((rows, vocab), generator=gen) * 3
    if kind == "peaks":
        x.scatter_add_(1, torch.randint(0, vocab, (rows, 5), generator=gen), torch.full((rows, 5), 15.0))
    elif kind == "equal":
        x[:] = 0.25
    elif kind == "rising":
        x[:] = torch.arange(vocab) / 64.0
    elif kind == "falling":
        x[:] = -torch.arange(vocab) / 64.0
    elif kind == "clump":                       # the largest side by side, all of them in few threads' shares
        x[:, vocab // 3:vocab // 3 + 300] += 40.0
    elif kind == "strided":                     # the largest at multiples of powers of two
        x[:, ::256] += 40.0
        x[:, ::1024] += 10.0
    elif kind == "few":                         # a vocabulary masked down to a few tokens
        keep = x[:, :3].clone()
        x[:] = -math.inf
        x[:, vocab // 2:vocab // 2 + 3] = keep[:, :min(3, vocab - vocab // 2)]
    elif kind == "lowest":                      # masked by the type's lowest value
        x[:, 1:] = torch.finfo(torch.float32).min
    elif kind == "zeros":                       # +0 and -0 are one value
        x[:] = torch.where(torch.rand((rows, vocab), generator=gen) < 0.5, 0.0, -0.0)
    elif kind == "coarse":                      # many equal ones
        x = x.round()
    return x


@pytest.mark.parametrize("rows,vocab,pad,n,top,dtype", [
    (1, 1, 0, 1, 1, F32), (3, 7, 2, 8, 7, F32), (2, 64, 0, 1, 64, BF16), (5, 1000, 3, 2, 20, F32), (4, 1025, 0, 3, 128, F32),
    (2, 4097, 1, 1, 5, BF16), (3, 16384, 0, 1, 5, F32), (3, 16385, 0, 4, 31, F32), (1, 65536, 0, 1, 5, F32), (2, 65536, 0, 0, 0, F32),
    (33, 65536, 0, 2, 33, F32), (1, 200003, 0, 5, 128, F32), (7, 100003, 5, 4, 8, BF16), (300, 5003, 1, 1, 1, BF16), (1030, 130, 0, 1, 3, F32),
    (2, 65536, 8, 8, 65, BF16), (600, 40001, 0, 1, 10, BF16)])
def test_logprobs_sizes(rows, vocab, pad, n, top, dtype):
    gen = torch.Generator().manual_seed(rows * 31 + vocab)
    wide = rows_of("peaks", rows, vocab + pad, gen).to(dtype).cuda()
    tokens = torch.randint(0, vocab, (rows, n), generator=gen, dtype=torch.int32).cuda() if n else None
    check_logprobs(wide[:, :vocab], tokens, top)
    if pad:
        check_logprobs(wide[:, pad:], tokens, top)             # rows that begin off every boundary
    if n == 1:
        got = ops.token_logprobs(wide[:, :vocab], tokens[:, 0].contiguous())
        assert got.logprobs.shape == (rows,) and got.ranks.shape == (rows,) and got.top_ids.shape == (rows, 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "clump", "strided", "few", "lowest", "zeros", "coarse"])
@pytest.mark.parametrize("vocab", [700, 20001, 70000])
def test_logprobs_values(kind, vocab, dtype):
    gen = torch.Generator().manual_seed(vocab)
    x = rows_of(kind, 3, vocab, gen).to(dtype).cuda()
    tokens = torch.randint(0, vocab, (3, 6), generator=gen, dtype=torch.int32)
    tokens[:, 0], tokens[:, 1], tokens[:, 2] = 0, vocab - 1, vocab // 2
    for top in (1, 7, 128):
        check_logprobs(x, tokens.cuda(), top)


@pytest.mark.parametrize("vocab", [5, 3000, 70001])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprobs_of_no_distribution(vocab, dtype):
    gen = torch.Generator().manual_seed(3)
    x = rows_of("random", 8, vocab, gen)
    x[1, vocab - 1] = math.nan
    x[2, 0] = -math.nan
    x[3, vocab // 2] = math.inf
    x[4] = -math.inf
    x[5, 0], x[5, 1] = math.inf, math.nan
    x[6, :] = math.nan
    x[7, 1:3] = math.inf
    tokens = torch.tensor([[0, vocab // 2, vocab - 1, -1, vocab, 2 ** 31 - 1, -2 ** 31]] * 8, dtype=torch.int32)
    check_logprobs(x.to(dtype).cuda(), tokens.cuda(), min(vocab, 4))


def test_logprobs_broadcast_and_empty():
    gen = torch.Generator().manual_seed(4)
    x = rows_of("peaks", 1, 33000, gen).cuda()
    tokens = torch.randint(0, 33000, (9, 2), generator=gen, dtype=torch.int32).cuda()
    check_logprobs(x.expand(9, 33000), tokens, 4)
    empty = ops.token_logprobs(x[:0], tokens[:0], top=3)
    assert empty.logprobs.shape == (0, 2) and empty.top_ids.shape == (0, 3) and empty.entropy.shape == (0,)


def test_logprobs_sum_to_one():
    x = (torch.randn((4, 100), generator=torch.Generator().manual_seed(5)) * 4).cuda()
    got = ops.token_logprobs(x, top=100)
    assert (got.top_logprobs.double().exp().sum(1) - 1).abs().max() < 1e-5
    assert torch.equal(got.top_ids.sort(1).values, torch.arange(100, dtype=torch.int32, device="cuda").expand(4, 100))


# ------------------------------------------------------------------------------------------------ attention of trees


def tree_of(kind, n, rng):
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "roots":
        return [-1] * n
    if kind == "invalid":                      # cycles, own indices, later ones, far ones: all of them roots
        return [rng.choice([i, i + 1, 2 ** 31 - 1, -2 ** 31, -7, max(0, i - 1), 0]) for i in range(n)]
    return [-1 if i == 0 else rng.randint(max(0, (i - 1) // 3), i - 1) for i in range(n)]


class Trees:
    """Requests with contexts and trees; pages in a random order; what no node may see is NaN or infinite."""

    def __init__(self, contexts, nodes, heads, kv_heads, dim, dtype, page=16, layers=2, kind="random", seed=0, width=None):
        rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
        self.page, self.layer = page, layers - 1
        counts = [-(-(c + n) // page) for c, n in zip(contexts, nodes)]
        n_pages = sum(counts) + 3
        order = list(range(n_pages))
        rng.shuffle(order)
        self.k = torch.full((n_pages, layers, kv_heads, page, dim), math.nan)
        self.v = torch.full((n_pages, layers, kv_heads, dim, page), math.nan)
        self.v[:, :, :, ::3] = math.inf
        width = width or max(counts) + 2
        self.table = torch.full((len(contexts) + 1, width), -1, dtype=torch.int32)
        used, parents = 0, []
        for r, (c, n) in enumerate(zip(contexts, nodes)):
            mine = order[used:used + counts[r]]
            used += counts[r]
            self.table[r, :counts[r]] = torch.tensor(mine, dtype=torch.int32)
            for p in range(c + n):
                at, off = mine[p // page], p % page
                self.k[at, :, :, off] = torch.randn((layers, kv_heads, dim), generator=gen)
                self.v[at, :, :, :, off] = torch.randn((layers, kv_heads, dim), generator=gen)
            parents += tree_of(kind, n, rng)
        self.k, self.v = self.k.to(dtype), self.v.to(dtype)
        self.slots, self.starts, self.parents = list(range(len(contexts))), list(contexts), parents
        self.offsets = [0]
        for n in nodes:
            self.offsets.append(self.offsets[-1] + n)
        self.rows = self.offsets[-1]
        self.q = (torch.randn((self.rows + 2, heads * dim), generator=gen) * 1.5).to(dtype)      # (two rows of no request)
        self.parents += [-1, 0]

    def run(self, window=0, scale=None, max_nodes=None, max_context=0, q=None, out=None):
        ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
        cache = ops.PagedCache(self.k.cuda(), self.v.cuda(), self.table.cuda())
        q = self.q.cuda() if q is None else q
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if out is None else out
        return ops.tree_attention(q, cache, self.layer, ints(self.slots), ints(self.starts), ints(self.offsets), ints(self.parents),
                                  scale=scale, window=window, max_nodes=max_nodes, max_context=max_context, out=out)

    def check(self, window=0, scale=None, max_nodes=None, max_context=0, only=None):
        got = self.run(window, scale, max_nodes, max_context).cpu()
        dim = self.k.shape[4]
        want, slack = plain.tree_attention(self.q, self.k, self.v, self.table, self.layer, self.slots, self.starts, self.offsets,
                                           self.parents, dim ** -0.5 if scale is None else scale, window, max_nodes or 256)
        mine = ~want.isnan()
        if only is None:
            assert (got[~mine] == 7.0).all()               # rows of no request stay as they were
        else:
            mine &= torch.tensor(only)[:, None]
        assert mine.any()
        error = (got.double() - want)[mine].abs()
        assert (error <= slack[mine] + plain.HALF_STEP[self.q.dtype] * (want[mine].abs() + slack[mine])).all(), error.max()
        return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (8, 1, 128), (3, 3, 32), (6, 2, 96), (16, 2, 64)])
@pytest.mark.parametrize("contexts,nodes", [((0,), (1,)), ((1, 17), (1, 5)), ((63, 64, 65, 200), (1, 16, 17, 3)), ((300, 0, 5), (33, 0, 64))])
def test_tree_sizes(contexts, nodes, heads, kv_heads, dim, dtype):
    Trees(contexts, nodes, heads, kv_heads, dim, dtype, seed=sum(contexts) + dim).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "invalid"])
@pytest.mark.parametrize("window", [0, 1, 2, 50])
def test_tree_shapes(kind, window, dtype):
    Trees((70, 3), (40, 9), 4, 2, 64, dtype, kind=kind, seed=3).check(window=window)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [255, 256])
def test_tree_of_many_nodes(n, dtype):
    for kind, window in (("chain", 0), ("random", 0), ("chain", 100)):
        Trees((37,), (n,), 2, 1, 64, dtype, kind=kind, seed=n).check(window=window)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page,dim", [(12, 64), (8, 64), (32, 64), (128, 64), (16, 40), (16, 256), (16, 7), (16, 160)])
def test_tree_pages_and_heads(page, dim, dtype):
    Trees((100, 31), (5, 20), 4, 2, dim, dtype, page=page, seed=dim).check(window=0 if page != 32 else 60)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tree_long_context(dtype):
    t = Trees((5000, 2100), (3, 6), 4, 1, 64, dtype, layers=1, seed=8, width=700)
    for hint in (0, 1, 5000, 1 << 30):
        t.check(max_context=hint)
    t.check(window=1000)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tree_scales(dtype):
    t = Trees((40,), (9,), 4, 2, 64, dtype, seed=9)
    for scale in (0.0, -0.3, 2.0):
        t.check(scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tree_single_tokens_are_decode(dtype):
    t = Trees((130, 64, 0, 15), (1, 1, 1, 1), 8, 2, 64, dtype, seed=10)
    t.check(max_nodes=1)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tree_of_what_is_not_seen(dtype):
    """Keys and values of one branch are NaN and infinite: the other branches do not notice."""
    t = Trees((20,), (30,), 4, 2, 64, dtype, kind="star", seed=11)
    for node, bad in ((3, math.nan), (17, math.inf), (29, -math.inf)):
        page = int(t.table[0, (20 + node) // 16])
        t.k[page, :, :, (20 + node) % 16] = bad
        t.v[page, :, :, :, (20 + node) % 16] = bad
    t.check(only=[i < 30 and i not in (3, 17, 29) for i in range(32)])
    # and in a window: the places before it
    t = Trees((100,), (4,), 4, 2, 64, dtype, kind="chain", seed=12)
    page = int(t.table[0, 80 // 16])
    t.v[page, :, :, :, :4] = math.nan                   # places 80 to 83
    t.check(window=17, only=[i < 4 for i in range(6)])
    t.check(window=20, only=[i == 3 for i in range(6)])     # node 3 stands at 103: 84 and later


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tree_slots_and_pages_outside(dtype):
    t = Trees((50, 60, 70), (4, 5, 6), 4, 2, 64, dtype, seed=13)
    t.slots[1] = 99
    t.check()
    t.slots[1] = -1
    t.check()
    t = Trees((200, 60), (4, 5), 4, 2, 64, dtype, seed=14)
    t.table[0, 2], t.table[0, 5], t.table[1, 0] = -1, 10 ** 6, -2 ** 31      # pages that are none: their keys are not seen
    t.check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("context,nodes", [(20, 3), (2000, 5), (300, 60)])
def test_tree_rows_that_see_nothing(context, nodes, page, dtype):
    t = Trees((context, 40), (nodes, 4), 8, 2, 64, dtype, layers=1, page=page, seed=17)
    t.table[0] = -1                                     # (the request has rows, and no page)
    got = t.check(max_context=context)
    assert (got[:nodes] == 0).all() and (got[nodes:nodes + 4] != 0).any()
    t = Trees((context,), (nodes,), 8, 2, 64, dtype, layers=1, page=page, seed=18, width=-(-(context + nodes) // page))
    t.starts[0] = t.table.shape[1] * page + 7           # all of the tree, and with the window what it sees, behind the table
    got = t.check(window=5)
    assert (got[:nodes] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page,nodes", [(16, 4), (16, 40), (12, 4)])
def test_tree_lists_that_name_anything(page, nodes, dtype):
    """Offsets that end before they begin or behind the rows, starts at both ends of the numbers: nothing but the request's own rows
    is written."""
    for bad in (-2 ** 31, -1, 2 ** 31 - 1):
        t = Trees((30, 40), (nodes, 5), 8, 2, 64, dtype, page=page, seed=19)
        t.offsets[1] = bad                              # the first request's end, the second's beginning
        got = t.run(max_nodes=nodes).cpu()
        assert (got[t.offsets[2]:] == 7.0).all() if bad < 0 else got.isfinite().all()
        t = Trees((30, 40), (nodes, 5), 8, 2, 64, dtype, page=page, seed=19)
        want = t.run(max_nodes=nodes).cpu()
        t.starts[0] = bad
        for window in (0, 9):
            got = t.run(max_nodes=nodes, window=window).cpu()
            assert (got[t.rows:] == 7.0).all()
            if not window:
                assert torch.equal(got[nodes:nodes + 5], want[nodes:nodes + 5])


def test_tree_rows_of_a_request_behind_max_nodes():
    t = Trees((30, 20), (9, 3), 4, 2, 64, BF16, seed=15)
    t.check(max_nodes=5)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tree_strided_queries(dtype):
    t = Trees((90,), (11,), 4, 2, 64, dtype, seed=16)
    want = t.run()
    for extra in (8, 3):
        wide = torch.zeros((t.q.shape[0], 256 + extra), dtype=dtype, device="cuda")
        wide[:, extra:] = t.q.cuda()
        assert torch.equal(t.run(q=wide[:, extra:]), want) or (t.run(q=wide[:, extra:]).float() - want.float()).abs().max() < 0.03


# ------------------------------------------------------------------------------------------------ tokens and pages


def cache_of(n_pages, layers, kv_heads, page, dim, v_dim, dtype, seed, slots, width):
    gen, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    k = torch.randn((n_pages, layers, kv_heads, page, dim), generator=gen).to(dtype)
    v = torch.randn((n_pages, layers, kv_heads, v_dim, page), generator=gen).to(dtype) if v_dim else None
    order = list(range(n_pages))
    rng.shuffle(order)
    table = torch.tensor(order[:slots * width], dtype=torch.int32).view(slots, width)
    return k, v, table


def moved(k, v, table, src, dst, offsets, places, starts):
    """Token by token, read from the old cache."""
    page, new_k, new_v = k.shape[3], k.clone(), None if v is None else v.clone()
    for r in range(len(src)):
        for i, p in enumerate(places[offsets[r]:offsets[r + 1]]):
            to = starts[r] + i
            if not (0 <= src[r] < table.shape[0] and 0 <= dst[r] < table.shape[0]):
                continue
            if p < 0 or to < 0 or p >= table.shape[1] * page or to >= table.shape[1] * page:
                continue
            a, b = int(table[src[r], p // page]), int(table[dst[r], to // page])
            if not (0 <= a < k.shape[0] and 0 <= b < k.shape[0]):
                continue
            new_k[b, :, :, to % page] = k[a, :, :, p % page]
            if v is not None:
                new_v[b, :, :, :, to % page] = v[a, :, :, :, p % page]
    return new_k, new_v


def check_move(k, v, table, src, dst, offsets, places, starts):
    want_k, want_v = moved(k, v, table, src, dst, offsets, places, starts)
    gk, gv, gt = k.cuda(), None if v is None else v.cuda(), table.cuda()
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    ops.move_tokens(ops.PagedCache(gk, gv, gt), ints(src), ints(dst), ints(offsets), ints(places), ints(starts))
    assert torch.equal(gk.cpu(), want_k)
    if v is not None:
        assert torch.equal(gv.cpu(), want_v)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page,dim,v_dim", [(16, 64, 64), (8, 32, 48), (32, 128, 128), (12, 40, 40), (16, 64, 0), (1, 7, 3), (64, 96, 96)])
def test_move_tokens(page, dim, v_dim, dtype):
    rng = random.Random(page + dim)
    width = -(-400 // page)
    k, v, table = cache_of(4 * width + 2, 3, 2, page, dim, v_dim, dtype, page * dim, 4, width)
    tail = sorted(rng.sample(range(200, 300), 60))
    # in place: a path moved up, every second token of a long stretch, and nothing at all; between slots: any order, with repeats
    check_move(k, v, table, [0, 1, 2], [0, 1, 2], [0, 60, 260, 260], tail + list(range(0, 400, 2)), [200, 0, 17])
    check_move(k, v, table, [0, 1], [0, 1], [0, 5, 6], [100, 101, 102, 120, 121, 7], [100, 7])           # (some stay where they are)
    check_move(k, v, table, [0, 0], [2, 3], [0, 100, 350], [rng.randrange(400) for _ in range(350)], [3, 150])
    check_move(k, v, table, [3], [1], [0, 400], list(range(399, -1, -1)), [0])
    check_move(k, v, table, [3], [1], [0, 1], [399], [399])


def test_move_tokens_leaves_out_what_is_not_there():
    k, v, table = cache_of(20, 2, 2, 16, 64, 64, BF16, 5, 3, 6)
    table[1, 2], table[2, 0], table[2, 1] = -1, 10 ** 6, -2 ** 31
    check_move(k, v, table, [0, 5, 0, -1], [1, 1, 7, 1], [0, 60, 61, 62, 63], list(range(30, 90)) + [1, 2, 3], [0, 90, 0, 91])
    check_move(k, v, table, [2], [0], [0, 40], list(range(40)), [20])
    check_move(k, v, table, [0], [1], [0, 6], [-1, 95, 96, 2 ** 31 - 1, -2 ** 31, 3], [85])
    check_move(k, v, table, [0], [1], [0, 4], [1, 2, 3, 4], [94])


def test_move_tokens_lists_that_name_anything():
    k, v, table = cache_of(20, 2, 2, 16, 64, 64, BF16, 5, 3, 6)
    for bad in (-2 ** 31, -1, 2 ** 31 - 1):
        gk, gv = k.cuda(), v.cuda()
        ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
        cache = ops.PagedCache(gk, gv, table.cuda())
        ops.move_tokens(cache, ints([0, 1]), ints([2, 2]), ints([3, bad, 3]), ints([1, 2, 3, 4]), ints([0, 40]))
        if bad < 0:                                     # (the first request has nothing; the second's entries begin at 0)
            want = moved(k, v, table, [1], [2], [0, 3], [1, 2, 3], [40])
        else:                                           # (the first one's entries end with the list)
            want = moved(k, v, table, [0], [2], [0, 1], [4], [0])
        assert torch.equal(gk.cpu(), want[0]) and torch.equal(gv.cpu(), want[1])


def test_a_cache_whose_tensors_moved():
    k, v, table = (x.cuda() for x in cache_of(4, 1, 1, 16, 32, 32, BF16, 6, 1, 4))
    cache, one = ops.PagedCache(k, v, table), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.copy_pages(cache, one, one)
    cache.v = v.clone()
    with pytest.raises(ValueError, match="moved"):
        ops.copy_pages(cache, one, one)


def test_move_tokens_many_in_place():
    """Thousands of tokens moved over each other, a few places up at a time."""
    k, v, table = cache_of(520, 2, 2, 16, 64, 64, BF16, 6, 1, 512)
    check_move(k, v, table, [0], [0], [0, 8000], list(range(3, 8003)), [0])
    check_move(k, v, table, [0], [0], [0, 4000], [2 * i + (i % 2) for i in range(4000)], [0])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page,dim,v_dim,kv_heads,layers", [(16, 64, 64, 8, 6), (1, 7, 3, 1, 1), (8, 32, 0, 2, 1), (12, 5, 9, 3, 2)])
def test_copy_pages(page, dim, v_dim, kv_heads, layers, dtype):
    k, v, table = cache_of(40, layers, kv_heads, page, dim, v_dim, dtype, 7, 1, 1)
    src, dst = [3, 39, 3, 7, -1, 5, 40, 6, 2 ** 31 - 1, 8], [0, 1, 2, 38, 20, 40, 21, -2 ** 31, 22, 8]
    want_k, want_v = k.clone(), None if v is None else v.clone()
    for a, b in zip(src, dst):
        if 0 <= a < 40 and 0 <= b < 40:
            want_k[b] = k[a]
            if v is not None:
                want_v[b] = v[a]
    gk, gv = k.cuda(), None if v is None else v.cuda()
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    cache = ops.PagedCache(gk, gv, table.cuda())
    ops.copy_pages(cache, ints(src), ints(dst))
    ops.copy_pages(cache, ints([]), ints([]))
    assert torch.equal(gk.cpu(), want_k)
    if v is not None:
        assert torch.equal(gv.cpu(), want_v)


# ------------------------------------------------------------------------------------------------ streams and graphs


def test_recorded_and_on_another_stream():
    """All four recorded into one graph, replayed with new inputs in the same memory between eager work."""
    t = Trees((90, 700), (12, 7), 8, 2, 64, BF16, seed=20)
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    k, v, table = t.k.cuda(), t.v.cuda(), t.table.cuda()
    cache = ops.PagedCache(k, v, table)
    q, logits = t.q.cuda(), torch.randn((30, 70001), device="cuda")
    tokens = torch.randint(0, 70001, (30, 2), device="cuda", dtype=torch.int32)
    slots, starts, offsets, parents = ints(t.slots), ints(t.starts), ints(t.offsets), ints(t.parents)
    kept_offsets, places = ints([0, 3, 5]), ints([90, 95, 99, 700, 704])
    spare = [p for p in range(k.shape[0]) if p not in t.table.flatten().tolist()]
    src, dst = ints([int(t.table[0, 0])]), ints(spare[:1])

    def work():
        a = ops.tree_attention(q, cache, 1, slots, starts, offsets, parents, max_nodes=12, max_context=700)
        b = ops.token_logprobs(logits, tokens, top=5)
        ops.copy_pages(cache, src, dst)
        ops.move_tokens(cache, slots, slots, kept_offsets, places, starts)
        return (a,) + tuple(b)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for turn in range(4):
        k.copy_(t.k), v.copy_(t.v)
        q.normal_(), logits.normal_().mul_(3)
        graph.replay()
        torch.cuda.synchronize()
        got, got_k, got_v = [o.clone() for o in out], k.clone(), v.clone()
        k.copy_(t.k), v.copy_(t.v)
        want = work()
        torch.cuda.synchronize()
        rows = t.rows
        assert torch.equal(got[0][:rows], want[0][:rows])
        for g, w in zip(got[1:], want[1:]):
            assert torch.equal(g, w)
        assert torch.equal(got_k.view(torch.int16), k.view(torch.int16)) and torch.equal(got_v.view(torch.int16), v.view(torch.int16))


def test_same_call_twice_gives_the_same_bits():
    t = Trees((1500,), (20,), 8, 2, 64, BF16, seed=21)
    assert torch.equal(t.run(), t.run())
    x = torch.randn((3, 90001), device="cuda")
    a, b = ops.token_logprobs(x, top=50), ops.token_logprobs(x, top=50)
    assert all(torch.equal(p, q) for p, q in zip(a[2:], b[2:]))


# ------------------------------------------------------------------------------------------------ used together


def test_draft_judge_keep_and_go_on():
    """A drafted tree is attended to, its path judged and kept; the request then goes on as if it had been fed the path alone."""
    dim, heads, kv_heads, vocab = 64, 4, 2, 500
    gen = torch.Generator().manual_seed(30)
    context, tree = 45, [-1, 0, 0, 1, 1, 2, 4, 4, 6]
    t = Trees((context,), (len(tree),), heads, kv_heads, dim, F32, seed=30, width=8)
    t.parents = tree + [-1, 0]
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    k, v, table = t.k.cuda(), t.v.cuda(), t.table.cuda()
    cache = ops.PagedCache(k, v, table)
    q = t.q.cuda()
    one = ints([0])
    out = ops.tree_attention(q, cache, 1, one, ints([context]), ints([0, len(tree)]), ints(t.parents), max_nodes=9)
    head = torch.randn((heads * dim, vocab), generator=gen).cuda()
    children = ints([[1, 2], [3, 4], [5, -1], [-1, -1], [6, 7], [-1, -1], [8, -1], [-1, -1], [-1, -1]])       # (a draft's token is its index here)
    judged = ops.token_logprobs(out[:9] @ head, children, top=3)
    assert torch.equal(judged.logprobs.isnan(), children < 0)
    # the path that the scoring model likes best, a node at a time
    path, at = [0], 0
    while (children[at] >= 0).any():
        at = int(children[at][judged.logprobs[at].nan_to_num(-math.inf).argmax()])
        path.append(at)
    before = out[path[-1]].clone()
    ops.move_tokens(cache, one, one, ints([0, len(path)]), ints([context + p for p in path]), ints([context]))
    # the last accepted node again, as a single token behind the kept ones
    row = q[path[-1]:path[-1] + 1]
    again = ops.tree_attention(row, cache, 1, one, ints([context + len(path) - 1]), ints([0, 1]), ints([-1]), max_nodes=1)
    assert (again[0] - before).abs().max() < 1e-5
    # a fork: the request's last page copied for a second one that shares the others
    pages = -(-(context + len(path)) // 16)
    spare = [p for p in range(k.shape[0]) if p not in t.table.flatten().tolist()][0]
    table[1] = table[0]
    table[1, pages - 1] = spare
    ops.copy_pages(cache, table[0, pages - 1:pages].contiguous(), ints([spare]))
    both = ops.tree_attention(row.repeat(2, 1), cache, 1, ints([0, 1]), ints([context + len(path) - 1] * 2), ints([0, 1, 2]), ints([-1, -1]),
                              max_nodes=1)
    assert torch.equal(both[0], both[1])
