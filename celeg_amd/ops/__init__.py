"""Operators on torch tensors for requests that go on in several ways, as a program calls them between a model's steps:

* ``token_logprobs``: log probabilities and ranks of given tokens, entropy, best alternatives, from rows of logits;
* ``tree_attention``: a tree of drafted tokens over its request's cached context;
* ``move_tokens``: cached tokens brought together (the accepted path of a tree, the kept tokens of a long context);
* ``copy_pages``: whole pages copied (a request that forks).

Thin callers of the library's C interface (``csrc/include/celeg_amd.h``, which says what each computes and refuses; the
kernels are ``csrc/token_logprobs.hip``, ``csrc/tree_attention.hip`` and ``csrc/cache_copy.hip``).  They run on torch's
current stream of the tensors' device and can be recorded into a graph; results and workspaces are torch's memory, so that nothing is
shared between calls.  A refused argument is a ``NativeArgumentError`` (a ``ValueError``)."""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from .. import native
from ..native import NativeArgumentError

MAX_TOKENS_PER_ROW = 8
MAX_TOP = 128
MAX_TREE_NODES = 256
_MAX_REQUEST_NODES = 65535       # requests times nodes of a call of the library

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _refuse(message: str):
    raise NativeArgumentError(message)


def _device(t: torch.Tensor, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(f"{name} must be a GPU tensor")
    return t.device


def _ints(t: torch.Tensor, name: str, count: Optional[int], device: torch.device) -> int:
    """The address of a list of 32-bit integers on the device."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.device != device or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous int32 tensor on {device}")
    if count is not None and t.numel() != count:
        _refuse(f"{name} must have {count} entries, not {t.numel()}")
    return t.data_ptr()


def _call(device: torch.device, function, *args) -> None:
    """function(*args, stream) with the tensors' device as the current one."""
    if device.index == torch.cuda.current_device():
        native.check(function(*args, _raw_stream(device.index)))
    else:
        with torch.cuda.device(device):
            native.check(function(*args, _raw_stream(device.index)))


class PagedCache:
    """All layers of one group of pages: ``k`` [pages, layers, kv_heads, page_tokens, head_dim], ``v`` [pages, layers, kv_heads,
    v_head_dim, page_tokens] (``None``: keys only), ``table`` int32 [slots, pages of a request].  The tensors are kept, not copied."""

    def __init__(self, k: torch.Tensor, v: Optional[torch.Tensor], table: torch.Tensor):
        self.device = _device(k, "k")
        if k.dim() != 5 or k.dtype not in _DTYPES or not k.is_contiguous():
            _refuse("k must be contiguous float32 or bfloat16 [pages, layers, kv_heads, page_tokens, head_dim]")
        if v is not None and (not isinstance(v, torch.Tensor) or v.dim() != 5 or v.dtype != k.dtype or v.device != k.device or
                              not v.is_contiguous() or v.shape[:3] != k.shape[:3] or v.shape[4] != k.shape[3]):
            _refuse("v must be contiguous [pages, layers, kv_heads, v_head_dim, page_tokens] of the keys' dtype and device")
        if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.dtype != torch.int32 or table.device != k.device or \
                not table.is_contiguous():
            _refuse("table must be contiguous int32 [slots, pages of a request] on the keys' device")
        self.k, self.v, self.table = k, v, table
        self.n_pages, self.n_layers, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        self.v_head_dim = v.shape[3] if v is not None else 0
        self.dtype = k.dtype
        self._struct = native.PagedCacheStruct(
            ctypes.sizeof(native.PagedCacheStruct), k.data_ptr(), v.data_ptr() if v is not None else None, table.data_ptr(),
            _DTYPES[k.dtype], self.n_pages, self.n_layers, self.kv_heads, self.page_tokens, self.head_dim, self.v_head_dim,
            table.shape[0], table.shape[1])
        self._ref = ctypes.byref(self._struct)

    def _here(self):
        """What the library is given, as long as the tensors are where they were."""
        s = self._struct
        if self.k.data_ptr() != s.k or (self.v is not None and self.v.data_ptr() != s.v) or self.table.data_ptr() != s.table:
            _refuse("the cache's tensors have moved: make a PagedCache of them anew")
        return self._ref


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]         # float32 [rows, n], shaped as the tokens were given (None: no tokens)
    ranks: Optional[torch.Tensor]            # int32, likewise
    entropy: torch.Tensor                    # float32 [rows]
    top_ids: torch.Tensor                    # int32 [rows, top]
    top_logprobs: torch.Tensor               # float32 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top: int = 0) -> TokenLogprobs:
    """``logits`` [rows, vocab], float32 or bfloat16, dense rows any distance apart; ``tokens`` int32 [rows] or [rows, n <= 8].
    A rank is the number of logits ahead of the token's (0: the most likely); alternatives come by (logit falling, index rising)."""
    device = _device(logits, "logits")
    if logits.dim() != 2 or logits.dtype not in _DTYPES:
        _refuse("logits must be float32 or bfloat16 [rows, vocab]")
    rows, vocab = logits.shape
    row_stride, column_stride = logits.stride()
    if column_stride != 1 and vocab > 1:
        _refuse("logits must have dense rows")
    per_row, address, logprobs, ranks = 0, None, None, None
    if tokens is not None:
        if not isinstance(tokens, torch.Tensor) or tokens.dim() not in (1, 2) or tokens.shape[0] != rows:
            _refuse("tokens must be int32 [rows] or [rows, n]")
        address = _ints(tokens, "tokens", None, device)
        per_row = tokens.shape[1] if tokens.dim() == 2 else 1
        # (sizes one by one: torch reads them faster than a tuple, 0.7 us a tensor)
        logprobs = torch.empty(*tokens.shape, dtype=torch.float32, device=device)
        ranks = torch.empty(*tokens.shape, dtype=torch.int32, device=device)
    if not 0 <= top <= MAX_TOP:
        _refuse(f"top must be in [0, {MAX_TOP}]")
    entropy = torch.empty(rows, dtype=torch.float32, device=device)
    top_ids = torch.empty(rows, top, dtype=torch.int32, device=device)
    top_logprobs = torch.empty(rows, top, dtype=torch.float32, device=device)
    args = native.TokenLogprobsArgs(
        ctypes.sizeof(native.TokenLogprobsArgs), logits.data_ptr(), rows, vocab, row_stride, _DTYPES[logits.dtype], per_row, top, address,
        logprobs.data_ptr() if per_row else None, ranks.data_ptr() if per_row else None, entropy.data_ptr(), top_ids.data_ptr(),
        top_logprobs.data_ptr())
    lib, ref, size = native.lib(), ctypes.byref(args), ctypes.c_size_t()
    native.check(lib.celeg_token_logprobs_workspace(ref, ctypes.byref(size)))
    workspace = torch.empty(size.value, dtype=torch.uint8, device=device) if size.value else None
    _call(device, lib.celeg_token_logprobs, ref, workspace.data_ptr() if size.value else None, size.value)
    return TokenLogprobs(logprobs, ranks, entropy, top_ids, top_logprobs)


def _attend(device: torch.device, args: native.TreeAttentionArgs, pages) -> None:
    lib, ref, size = native.lib(), ctypes.byref(args), ctypes.c_size_t()
    native.check(lib.celeg_tree_attention_workspace(ref, pages, ctypes.byref(size)))
    workspace = torch.empty(size.value, dtype=torch.uint8, device=device) if size.value else None
    _call(device, lib.celeg_tree_attention, ref, pages, workspace.data_ptr() if size.value else None, size.value)


def tree_attention(q: torch.Tensor, cache: PagedCache, layer: int, slots: torch.Tensor, starts: torch.Tensor, offsets: torch.Tensor,
                   parents: torch.Tensor, *, scale: Optional[float] = None, window: int = 0, max_nodes: Optional[int] = None,
                   max_context: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of ``q`` [rows, heads * head_dim] (dense rows, the cache's dtype) are the nodes of the requests' trees, request r's the rows
    ``offsets[r]`` to ``offsets[r + 1] - 1``; their keys and values lie in ``cache`` behind the request's context, node i's at place
    ``starts[r] + i`` of slot ``slots[r]``.  ``parents[row]``: the parent's index inside the tree, -1 for a root.  A node sees the
    context, its ancestors and itself (with a ``window``: fewer than so many positions back).  ``scale`` defaults to
    head_dim ** -0.5; ``max_nodes`` is the most nodes of a request (default: the rows, at most 256: of many requests it is worth saying,
    as the work is cut by it; 1 where every request brings a single token), ``max_context`` about the longest context (0: what the
    table holds), by which the work is cut.  ``out`` [rows, heads * head_dim] is
    made if it is not given; rows of no request are then undefined, and left as they were where it is."""
    if not isinstance(cache, PagedCache):
        _refuse("cache must be a PagedCache")
    device = cache.device
    if not isinstance(q, torch.Tensor) or q.device != device or q.dtype != cache.dtype or q.dim() != 2:
        _refuse("q must be [rows, heads * head_dim] of the cache's dtype and device")
    rows, width = q.shape
    q_stride, column_stride = q.stride()
    if column_stride != 1 and width > 1:
        _refuse("q must have dense rows")
    if width == 0 or width % cache.head_dim:
        _refuse("the width of q must be a multiple of the cache's head_dim")
    if out is None:
        out = torch.empty(rows, width, dtype=q.dtype, device=device)
    elif not isinstance(out, torch.Tensor) or out.device != device or out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous():
        _refuse("out must be contiguous, of q's shape, dtype and device")
    requests = slots.shape[0] if isinstance(slots, torch.Tensor) and slots.dim() == 1 else -1
    slots_at, starts_at = _ints(slots, "slots", requests, device), _ints(starts, "starts", requests, device)
    offsets_at, parents_at = _ints(offsets, "offsets", requests + 1, device), _ints(parents, "parents", rows, device)
    if max_nodes is None:
        max_nodes = min(max(rows, 1), MAX_TREE_NODES)
    args = native.TreeAttentionArgs(
        ctypes.sizeof(native.TreeAttentionArgs), q.data_ptr(), q_stride, out.data_ptr(), rows, width // cache.head_dim, requests, layer,
        slots_at, starts_at, offsets_at, parents_at, cache.head_dim ** -0.5 if scale is None else scale, window, max_nodes, max_context)
    if requests * max_nodes <= _MAX_REQUEST_NODES or max_nodes < 1:
        _attend(device, args, cache._here())
        return out
    # more requests than a call of the library takes: several, each with its part of the lists
    most = max(1, _MAX_REQUEST_NODES // max_nodes)
    for first in range(0, requests, most):
        args.requests = min(requests - first, most)
        args.slots, args.starts, args.offsets = slots_at + 4 * first, starts_at + 4 * first, offsets_at + 4 * first
        _attend(device, args, cache._here())
    return out


def move_tokens(cache: PagedCache, src_slots: torch.Tensor, dst_slots: torch.Tensor, offsets: torch.Tensor, places: torch.Tensor,
                dst_starts: torch.Tensor) -> None:
    """Keys and values of all layers: for every request r, the tokens at places ``places[offsets[r]:offsets[r + 1]]`` of slot
    ``src_slots[r]`` go to the places ``dst_starts[r]``, ``dst_starts[r] + 1``, .. of slot ``dst_slots[r]``.  Within one slot the places
    have to rise and no token may move up; between two, none that is read may lie where one is written (forked slots share pages). No place
    that a request writes may be one that another reads or writes."""
    if not isinstance(cache, PagedCache):
        _refuse("cache must be a PagedCache")
    device = cache.device
    if not isinstance(src_slots, torch.Tensor) or src_slots.dim() != 1:
        _refuse("src_slots must be int32 [requests]")
    if not isinstance(places, torch.Tensor) or places.dim() != 1:
        _refuse("places must be int32 [entries]")
    requests = src_slots.shape[0]
    _call(device, native.lib().celeg_move_tokens, cache._here(), requests, _ints(src_slots, "src_slots", requests, device),
          _ints(dst_slots, "dst_slots", requests, device), _ints(offsets, "offsets", requests + 1, device),
          _ints(places, "places", None, device), places.shape[0], _ints(dst_starts, "dst_starts", requests, device))


def copy_pages(cache: PagedCache, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Pages ``src[i]`` copied to ``dst[i]``, all layers.  No page may be written twice, or written and read."""
    if not isinstance(cache, PagedCache):
        _refuse("cache must be a PagedCache")
    if not isinstance(src, torch.Tensor) or src.dim() != 1:
        _refuse("src must be int32 [pairs]")
    n = src.shape[0]
    _call(cache.device, native.lib().celeg_copy_pages, cache._here(), _ints(src, "src", n, cache.device), _ints(dst, "dst", n, cache.device), n)


__all__ = ["PagedCache", "TokenLogprobs", "token_logprobs", "tree_attention", "move_tokens", "copy_pages", "MAX_TOKENS_PER_ROW",
           "MAX_TOP", "MAX_TREE_NODES"]
