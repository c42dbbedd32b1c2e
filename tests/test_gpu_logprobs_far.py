"""``ops.token_logprobs`` of logits far from 0: what counts is their distance from the row's largest, whatever that is."""
import math

import pytest
import torch

from celeg_amd import ops

import plain_branch as plain

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
LEVELS = [3e3, 1e6, 2.0 ** 24 - 4, 2.0 ** 24, 3e7, 1e9, 1e10, 1e20, 1e30, 3e38]


def rows_at(kind, level, rows, vocab, dtype, gen):
    x = torch.full((rows, vocab), level, dtype=torch.float64)
    if kind == "steps":              # the level and, in a few places, its neighbours in the type, up to three steps towards 0
        step = 2.0 ** (math.floor(math.log2(abs(level))) - (23 if dtype is F32 else 7))
        places = torch.randint(0, vocab, (rows, 9), generator=gen)
        x.scatter_(1, places, level - step * torch.randint(0, 4, (rows, 9), generator=gen).double() * math.copysign(1.0, level))
    elif kind == "masked":           # a vocabulary masked down to a few tokens by a number, these at the level
        x[:] = -1e30 if level > -1e30 else -3.2e38
        x.scatter_(1, torch.randint(0, vocab, (rows, 5), generator=gen), level)
    elif kind == "parts":            # the largest of one part far below another's
        x[:, :vocab // 2] = level / 2 if level > 0 else level * 2
    return x.to(torch.float32).to(dtype)


def check(x, tokens, top):
    got, want = ops.token_logprobs(x.cuda(), tokens.cuda(), top=top), plain.token_logprobs(x, tokens, top)
    vocab = x.shape[1]
    # An exponential's argument is rounded up to three times (a difference, a product, log2 e itself: 2.25 half steps of it), the
    # exponential to a step (2 half steps); weighed by their share the arguments are at most log2(vocab).  The sums: a thread adds up to
    # vocab / 256 terms one after the other (at most 64), or, from memory, up to 256, and the threads' and parts' sums are joined in fewer
    # than 64 more.  Their logarithm (a step of up to log2(vocab)) less what the maximum's rounding left out (1 at most), times ln 2: 4 more.
    near = 2.0 ** -24 * (min(vocab / 256, 256) + 64 + 2.25 * math.log2(vocab + 1) + 4 * math.log2(vocab + 1) + 8)
    for name, g, w in zip(got._fields, got, want):
        g = g.cpu()
        if g.dtype == torch.int32:
            assert torch.equal(g.long(), w), name
            continue
        assert not g.isnan().any() and torch.equal(g.isinf(), w.float().isinf()), name
        ok = w.float().isfinite()
        # (the entropy's terms are e d: the same relative errors of numbers up to the logarithm of the vocabulary)
        tolerance = near * (4 + math.log(vocab + 1)) if name == "entropy" else near + 2.0 ** -23 * w[ok].abs()
        assert ((g[ok].double() - w[ok]).abs() <= tolerance).all(), (name, (g[ok].double() - w[ok]).abs().max())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("kind", ["level", "steps", "masked", "parts"])
def test_logprobs_far_from_zero(kind, level, sign, dtype):
    for rows, vocab in ((3, 1000), (2, 20001), (2, 70001), (260, 17000)):
        gen = torch.Generator().manual_seed(vocab)
        x = rows_at(kind, sign * level, rows, vocab, dtype, gen)
        tokens = torch.randint(0, vocab, (rows, 3), generator=gen, dtype=torch.int32)
        tokens[:, 0] = x.float().argmax(1).int()
        check(x, tokens, 5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_logprobs_parts_on_both_sides_of_the_limit(sign, dtype):
    """The maxima of a row's parts lie below and above 2^24, where sums take their distances another way."""
    step = 1.0 if dtype is F32 else 2.0 ** 17
    for rows, vocab in ((2, 70001), (260, 33000)):
        gen = torch.Generator().manual_seed(vocab)
        near = torch.randint(-3, 3, (rows, vocab), generator=gen).double() * step + 2.0 ** 24
        x = (sign * near).to(torch.float32).to(dtype)
        tokens = torch.randint(0, vocab, (rows, 3), generator=gen, dtype=torch.int32)
        check(x, tokens, 5)


def test_logprobs_of_ordinary_logits_at_another_height():
    """A row moved by a constant that its type can hold says the same."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randint(-4096, 4096, (5, 33000), generator=gen).float() / 512          # multiples of 2^-9, up to 8
    tokens = torch.randint(0, 33000, (5, 4), generator=gen, dtype=torch.int32)
    here = ops.token_logprobs(x.cuda(), tokens.cuda(), top=8)
    for moved in (1024.0, -4096.0, 16376.0):                                         # (14 bits and 9 behind the point: exact)
        y = x + moved
        assert torch.equal(y - moved, x)
        check(y, tokens, 8)
        there = ops.token_logprobs(y.cuda(), tokens.cuda(), top=8)
        assert torch.equal(here.top_ids, there.top_ids) and torch.equal(here.ranks, there.ranks)
