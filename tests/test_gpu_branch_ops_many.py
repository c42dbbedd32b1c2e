"""``celeg_amd.ops`` with more requests, rows and pairs than one launch or one call of the library takes."""
import random

import pytest
import torch

from celeg_amd import ops

import plain_branch as plain
from test_gpu_branch_ops import Trees

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 40])
def test_trees_of_many_requests_without_a_bound_on_their_nodes(dim, dtype):
    """600 requests of which one has 200 nodes, most a few and some none: the rows alone do not say how many a request has."""
    rng = random.Random(dim)
    nodes = [rng.choice([0, 1, 1, 1, 2, 5]) for _ in range(600)]
    nodes[417] = 200
    t = Trees([rng.randint(0, 30) for _ in nodes], nodes, 4, 2, dim, dtype, layers=1, seed=dim)
    t.check()
    t.check(window=9)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [32, 24])
def test_trees_of_few_rows_among_very_many_requests_and_heads(dim, dtype):
    """65,535 requests, 256 key/value heads: more workgroups than a launch of the matrix-core kernel has."""
    gen = torch.Generator().manual_seed(dim)
    k, v = (torch.randn(s, generator=gen).to(dtype) for s in ((3, 1, 256, 16, dim), (3, 1, 256, dim, 16)))
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    requests, mine = 65535, (0, 40000, 65534)
    starts, offsets = [0] * requests, [0]
    for r in range(requests):
        offsets.append(offsets[-1] + (r in mine))
        starts[r] = 20 + mine.index(r) if r in mine else 0
    q = torch.randn((3, 256 * dim), generator=gen).to(dtype)
    ints = lambda x: torch.tensor(x, dtype=torch.int32)
    got = ops.tree_attention(q.cuda(), ops.PagedCache(k.cuda(), v.cuda(), table.cuda()), 0, ints([0] * requests).cuda(), ints(starts).cuda(),
                             ints(offsets).cuda(), ints([-1] * 3).cuda(), max_nodes=1, max_context=30).cpu().double()
    want, slack = plain.tree_attention(q, k, v, table, 0, [0] * 3, [starts[r] for r in mine], [0, 1, 2, 3], [-1] * 3, dim ** -0.5, 0, 1)
    assert ((got - want).abs() <= slack + plain.HALF_STEP[dtype] * (want.abs() + slack)).all()


def test_logprobs_of_more_rows_than_a_launch_has():
    """A second launch, with few rows of its own (which are cut otherwise)."""
    for rows, vocab in (((1 << 23) // 2 + 7, 1500), ((1 << 24) + 300, 3)):
        x = torch.randint(-8, 8, (64, vocab), generator=torch.Generator().manual_seed(vocab)).float() / 4
        wide = x.repeat((rows + 63) // 64, 1)[:rows].cuda() if vocab < 100 else None
        if wide is None:
            # (rows that lie on top of one another, as far as the operator allows: all of them the same one)
            wide = x[:1].cuda().expand(rows, vocab)
            x = x[:1]
        tokens = (torch.arange(rows, device="cuda", dtype=torch.int32) % vocab)[:, None].contiguous()
        got = ops.token_logprobs(wide, tokens, top=2)
        logp = torch.log_softmax(x.double(), 1).cuda()
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        place = torch.empty_like(order).scatter_(1, order, torch.arange(vocab).expand_as(order)).int().cuda()
        of = torch.arange(rows, device="cuda") % x.shape[0]
        for first in range(0, rows, 1 << 21):
            at, t = of[first:first + (1 << 21)], tokens[first:first + (1 << 21), 0].long()
            part = [g[first:first + (1 << 21)] for g in got]
            assert torch.equal(part[1][:, 0], place[at, t])
            assert torch.equal(part[3], order.cuda()[at, :2].int())
            # (a thread adds up to 16 exponentials, each and their sum rounded to a step, 2^-23 each; the logarithm of up to 1,500 to one of 11)
            assert (part[0][:, 0].double() - logp[at, t]).abs().max() <= 64 * 2.0 ** -23
            assert (part[4].double() - logp[at[:, None], part[3].long()]).abs().max() <= 64 * 2.0 ** -23
        entropy = -(logp.exp() * logp).sum(1)
        assert (got.entropy.double() - entropy[of]).abs().max() <= 256 * 2.0 ** -23
