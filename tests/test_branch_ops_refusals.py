"""What the operators of ``celeg_amd.ops`` refuse, without a GPU: every refusal comes before anything is launched."""
import ctypes

import pytest
import torch

from celeg_amd import native, ops

ADDRESS = 1 << 20         # never read: a refused call launches nothing


def cache(**changes):
    fields = dict(struct_size=ctypes.sizeof(native.PagedCacheStruct), k=ADDRESS, v=ADDRESS, table=ADDRESS, dtype=1, n_pages=9, n_layers=2,
                  kv_heads=2, page_tokens=16, head_dim=64, v_head_dim=64, table_rows=3, table_stride=4)
    fields.update(changes)
    return native.PagedCacheStruct(**fields)


def logprobs(**changes):
    fields = dict(struct_size=ctypes.sizeof(native.TokenLogprobsArgs), logits=ADDRESS, rows=2, vocab=100, row_stride=100, dtype=0, per_row=1,
                  top=5, tokens=ADDRESS, logprobs=ADDRESS, ranks=ADDRESS, entropy=ADDRESS, top_ids=ADDRESS, top_logprobs=ADDRESS)
    fields.update(changes)
    return native.TokenLogprobsArgs(**fields)


def tree(**changes):
    fields = dict(struct_size=ctypes.sizeof(native.TreeAttentionArgs), q=ADDRESS, q_stride=256, out=ADDRESS, rows=3, heads=4, requests=1,
                  layer=1, slots=ADDRESS, starts=ADDRESS, offsets=ADDRESS, parents=ADDRESS, scale=0.1, window=0, max_nodes=3, max_context=0)
    fields.update(changes)
    return native.TreeAttentionArgs(**fields)


def refused(function, *args):
    with pytest.raises(native.NativeArgumentError) as err:
        native.check(function(*args))
    assert str(err.value)
    return str(err.value)


@pytest.mark.parametrize("changes", [
    dict(struct_size=8), dict(dtype=2), dict(dtype=-1), dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(per_row=9), dict(per_row=-1),
    dict(top=129), dict(top=-1), dict(vocab=4, row_stride=4), dict(row_stride=99), dict(row_stride=-100), dict(logits=None), dict(tokens=None),
    dict(logprobs=None), dict(ranks=None), dict(top_ids=None), dict(top_logprobs=None)])
def test_logprobs(changes):
    a = logprobs(**changes)
    refused(native.lib().celeg_token_logprobs, ctypes.byref(a), ADDRESS, 1 << 40, None)


def test_logprobs_workspace():
    size = ctypes.c_size_t()
    for a in (logprobs(), logprobs(vocab=200000, row_stride=200000, top=128)):
        native.check(native.lib().celeg_token_logprobs_workspace(ctypes.byref(a), ctypes.byref(size)))
        if size.value:
            assert "workspace" in refused(native.lib().celeg_token_logprobs, ctypes.byref(a), ADDRESS, size.value - 1, None)
            assert "workspace" in refused(native.lib().celeg_token_logprobs, ctypes.byref(a), None, size.value, None)
            assert "workspace" in refused(native.lib().celeg_token_logprobs, ctypes.byref(a), ADDRESS + 4, size.value, None)
    refused(native.lib().celeg_token_logprobs_workspace, ctypes.byref(logprobs()), None)
    refused(native.lib().celeg_token_logprobs_workspace, None, ctypes.byref(size))


@pytest.mark.parametrize("changes", [
    dict(struct_size=8), dict(rows=-1), dict(requests=-1), dict(heads=0), dict(heads=3), dict(heads=-2), dict(max_nodes=0), dict(max_nodes=257),
    dict(requests=65535, max_nodes=2), dict(window=-1), dict(max_context=-1), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(q_stride=255), dict(q_stride=-1), dict(q_stride=1 << 31), dict(layer=2), dict(layer=-1), dict(q=None), dict(out=None), dict(slots=None),
    dict(starts=None), dict(offsets=None), dict(parents=None)])
def test_tree(changes):
    a, c = tree(**changes), cache()
    refused(native.lib().celeg_tree_attention, ctypes.byref(a), ctypes.byref(c), ADDRESS, 1 << 40, None)


CACHES = [dict(struct_size=8), dict(dtype=3), dict(k=None), dict(v=None), dict(v_head_dim=0), dict(table=None), dict(n_pages=0), dict(n_layers=0),
          dict(kv_heads=0), dict(page_tokens=0), dict(head_dim=0), dict(v_head_dim=-1), dict(table_rows=0), dict(table_stride=0),
          dict(table_stride=1 << 27), dict(n_layers=40000)]


@pytest.mark.parametrize("changes", CACHES + [dict(head_dim=257, v_head_dim=257), dict(v_head_dim=32), dict(v=None, v_head_dim=0)])
def test_tree_caches(changes):
    a, c = tree(q_stride=4096), cache(**changes)
    refused(native.lib().celeg_tree_attention, ctypes.byref(a), ctypes.byref(c), ADDRESS, 1 << 40, None)


def test_tree_workspace():
    size = ctypes.c_size_t()
    for a, c in ((tree(), cache()), (tree(rows=200, max_nodes=256, max_context=50000), cache(table_stride=4096, dtype=0))):
        native.check(native.lib().celeg_tree_attention_workspace(ctypes.byref(a), ctypes.byref(c), ctypes.byref(size)))
        if size.value:
            assert "workspace" in refused(native.lib().celeg_tree_attention, ctypes.byref(a), ctypes.byref(c), ADDRESS, size.value - 1, None)
            assert "workspace" in refused(native.lib().celeg_tree_attention, ctypes.byref(a), ctypes.byref(c), ADDRESS + 8, size.value, None)
    refused(native.lib().celeg_tree_attention_workspace, None, ctypes.byref(cache()), ctypes.byref(size))
    refused(native.lib().celeg_tree_attention_workspace, ctypes.byref(tree()), None, ctypes.byref(size))


@pytest.mark.parametrize("changes", CACHES)
def test_moves_and_copies(changes):
    c = cache(**changes)
    refused(native.lib().celeg_move_tokens, ctypes.byref(c), 1, ADDRESS, ADDRESS, ADDRESS, ADDRESS, 1, ADDRESS, None)
    refused(native.lib().celeg_copy_pages, ctypes.byref(c), ADDRESS, ADDRESS, 1, None)


def test_lists():
    c, lib = cache(), native.lib()
    refused(lib.celeg_move_tokens, ctypes.byref(c), -1, ADDRESS, ADDRESS, ADDRESS, ADDRESS, 1, ADDRESS, None)
    refused(lib.celeg_move_tokens, ctypes.byref(c), 1, ADDRESS, ADDRESS, ADDRESS, ADDRESS, -1, ADDRESS, None)
    for missing in range(5):
        lists = [ADDRESS] * 5
        lists[missing] = None
        refused(lib.celeg_move_tokens, ctypes.byref(c), 1, lists[0], lists[1], lists[2], lists[3], 1, lists[4], None)
    refused(lib.celeg_copy_pages, ctypes.byref(c), ADDRESS, ADDRESS, -1, None)
    refused(lib.celeg_copy_pages, ctypes.byref(c), None, ADDRESS, 1, None)
    refused(lib.celeg_copy_pages, ctypes.byref(c), ADDRESS, None, 1, None)


def test_addresses_off_their_types():
    lib, odd = native.lib(), ADDRESS + 1
    for name in ("logits", "tokens", "logprobs", "ranks", "entropy", "top_ids", "top_logprobs"):
        assert "boundar" in refused(lib.celeg_token_logprobs, ctypes.byref(logprobs(**{name: odd})), ADDRESS, 1 << 40, None)
    for name in ("q", "out", "slots", "starts", "offsets", "parents"):
        assert "boundar" in refused(lib.celeg_tree_attention, ctypes.byref(tree(**{name: odd})), ctypes.byref(cache()), ADDRESS, 1 << 40, None)
    for name in ("k", "v", "table"):
        assert "boundar" in refused(lib.celeg_copy_pages, ctypes.byref(cache(**{name: odd})), ADDRESS, ADDRESS, 1, None)
    for at in range(5):
        lists = [ADDRESS] * 5
        lists[at] = odd
        assert "boundar" in refused(lib.celeg_move_tokens, ctypes.byref(cache()), 1, lists[0], lists[1], lists[2], lists[3], 1, lists[4], None)
    assert "boundar" in refused(lib.celeg_copy_pages, ctypes.byref(cache()), ADDRESS, odd, 1, None)


def test_nothing_to_do():
    lib = native.lib()
    native.check(lib.celeg_token_logprobs(ctypes.byref(logprobs(rows=0, logits=None, tokens=None)), None, 0, None))
    native.check(lib.celeg_tree_attention(ctypes.byref(tree(rows=0, q=None)), ctypes.byref(cache()), None, 0, None))
    native.check(lib.celeg_tree_attention(ctypes.byref(tree(requests=0, slots=None)), ctypes.byref(cache()), None, 0, None))
    native.check(lib.celeg_move_tokens(ctypes.byref(cache()), 0, None, None, None, None, 1, None, None))
    native.check(lib.celeg_move_tokens(ctypes.byref(cache()), 1, None, None, None, None, 0, None, None))
    native.check(lib.celeg_copy_pages(ctypes.byref(cache()), None, None, 0, None))


def test_host_tensors():
    k, v = torch.zeros((2, 1, 1, 16, 64)), torch.zeros((2, 1, 1, 64, 16))
    with pytest.raises(ValueError):
        ops.PagedCache(k, v, torch.zeros((1, 2), dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros((2, 5)))
    for call in (lambda: ops.tree_attention(k, None, 0, k, k, k, k), lambda: ops.move_tokens(None, k, k, k, k, k), lambda: ops.copy_pages(None, k, k)):
        with pytest.raises(ValueError):
            call()
