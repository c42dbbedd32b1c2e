"""The operators of ``celeg_amd.ops`` in 64 bits on the CPU, from their definitions, with what the tests' tolerances are made of."""
import math

import torch

F64 = torch.float64
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # half the distance of neighbours, relative to the value


def token_logprobs(logits, tokens, top):
    """(logprobs, ranks, entropy, top_ids, top_logprobs) by the rules of the operator."""
    x = logits.detach().cpu().to(F64)
    rows, vocab = x.shape
    nan = x.isnan().any(1)
    high = x.amax(1) if vocab else x.new_zeros(rows)
    none = nan | (high == math.inf) | (high == -math.inf)
    high = torch.where(none, torch.zeros_like(high), high)
    d = x - high[:, None]
    e = torch.exp(d)
    total = e.sum(1)
    moment = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1)
    log_sum = torch.where(none, torch.full_like(total, math.nan), torch.log(total))
    entropy = log_sum - moment / total
    order = torch.sort(torch.where(nan[:, None], torch.zeros_like(x), x), dim=1, descending=True, stable=True).indices
    place = torch.empty_like(order).scatter_(1, order, torch.arange(vocab).expand(rows, vocab))
    logp = d - log_sum[:, None]
    logprobs = ranks = None
    if tokens is not None:
        t = tokens.detach().cpu().long().view(rows, -1)
        valid = (t >= 0) & (t < vocab)
        safe = t.clamp(0, vocab - 1)
        logprobs = torch.where(valid, logp.gather(1, safe), torch.full(t.shape, math.nan, dtype=F64)).view(tokens.shape)
        ranks = torch.where(valid & ~nan[:, None], place.gather(1, safe), -torch.ones_like(t)).view(tokens.shape)
    ids = order[:, :top]
    top_logprobs = logp.gather(1, ids)
    ids = torch.where(nan[:, None], -torch.ones_like(ids), ids)
    return logprobs, ranks, entropy, ids, top_logprobs


def paths(parents):
    """Every node's way up: itself, its parent, .. ; what is no index below a node's own ends the way."""
    out = []
    for i in range(len(parents)):
        at, way = i, [i]
        while 0 <= parents[at] < at:
            at = parents[at]
            way.append(at)
        out.append(way)
    return out


def tree_attention(q, k, v, table, layer, slots, starts, offsets, parents, scale, window, max_nodes):
    """(out, bound of the error beside the output's own rounding), rows of no request NaN.  All arguments on the CPU."""
    kv_heads, page, dim = k.shape[2], k.shape[3], k.shape[4]
    q64 = q.to(F64).view(q.shape[0], -1, dim)
    heads = q64.shape[1]
    out, slack = torch.full_like(q64, math.nan), torch.zeros_like(q64)
    half = HALF_STEP[k.dtype]
    for r in range(len(slots)):
        first, count = offsets[r], min(offsets[r + 1] - offsets[r], max_nodes)
        if not 0 <= slots[r] < table.shape[0]:
            continue
        pages = table[slots[r]].tolist()
        ways = paths(parents[first:first + count])
        for i in range(count):
            depth = len(ways[i]) - 1
            low = max(0, starts[r] + depth - window + 1) if window else 0
            places = list(range(low, starts[r])) + sorted(starts[r] + a for up, a in enumerate(ways[i]) if not window or up < window)
            places = [p for p in places if p // page < len(pages) and 0 <= pages[p // page] < k.shape[0]]
            where, at = (torch.tensor(x, dtype=torch.long) for x in ([pages[p // page] for p in places], [p % page for p in places]))
            for h in range(heads):
                kh = k[where, layer, h // (heads // kv_heads), at].to(F64)
                vh = v[where, layer, h // (heads // kv_heads), :, at].to(F64)
                qh = q64[first + i, h]
                score = kh @ qh * scale
                w = torch.softmax(score, 0)
                out[first + i, h] = w @ vh
                # a score is off by the roundings of dim sums of 32 bits and of the softmax's argument, a weight by that twice (its own
                # and the sum's); a weight in bfloat16 by half a step of it more; the sums over the keys by one of 32 bits each
                ds = ((dim + 8) * 2.0 ** -24 * abs(scale) * (kh.abs() @ qh.abs()).max() + 2.0 ** -22 * score.abs().max()) if len(places) else 0.0
                weight = 2 * ds + (half if k.dtype == torch.bfloat16 else 0.0) + (len(places) + 16) * 2.0 ** -24
                slack[first + i, h] = weight * (w @ vh.abs())
    return out.view(q.shape), slack.view(q.shape)
