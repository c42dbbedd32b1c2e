"""``ops.tree_attention`` again: queries whose rows lie any distance apart against 64 bits, and calls that repeat themselves to the bit."""
import pytest
import torch

from celeg_amd import ops

import plain_branch as plain
from test_gpu_branch_ops import Trees

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("extra", [8, 3])
def test_queries_any_distance_apart(extra, dtype):
    """(Rows on 16 bytes and off them: the matrix cores' kernel and the one for any sizes.)"""
    t = Trees((90, 7), (11, 40), 4, 2, 64, dtype, seed=16)
    wide = torch.full((t.q.shape[0], 256 + extra), float("nan"), dtype=dtype, device="cuda")
    wide[:, extra:] = t.q.cuda()
    got = t.run(q=wide[:, extra:]).cpu()
    want, slack = plain.tree_attention(t.q, t.k, t.v, t.table, t.layer, t.slots, t.starts, t.offsets, t.parents, 64 ** -0.5, 0, 256)
    mine = ~want.isnan()
    assert ((got.double() - want)[mine].abs() <= slack[mine] + plain.HALF_STEP[dtype] * (want[mine].abs() + slack[mine])).all()
    assert (got[~mine] == 7.0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("contexts,nodes,heads,kv_heads,dim", [
    ((700,), (8,), 16, 8, 64), ((3000, 1400), (26, 11), 32, 8, 64), ((4000, 2500), (64, 64), 8, 2, 128), ((9000,), (1,), 8, 2, 64), ((60,), (5,), 4, 2, 40)])
def test_calls_repeat_themselves(contexts, nodes, heads, kv_heads, dim, dtype):
    """Few rows, rows that share staged keys, long contexts in parts, single tokens, any sizes: nothing hangs on an order that may change."""
    t = Trees(contexts, nodes, heads, kv_heads, dim, dtype, layers=1, seed=dim)
    first = t.run(max_nodes=max(nodes))
    for _ in range(5):
        junk = torch.full((1 << 20,), float("nan"), device="cuda")       # (what a workspace may find in its memory)
        del junk
        assert torch.equal(t.run(max_nodes=max(nodes)), first)
