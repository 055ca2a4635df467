"""Drafted trees in a ragged batch on a paged KV cache: a step checks many guessed
tokens of each request at once and keeps the way that the model itself chose.

* ``DraftTree.encode_plan``    parents -> positions and ancestors of every node
* ``TreeAttention.encode``     attention of the nodes over prefix, history and ancestors
* ``DraftAccept.encode``       the walk down each tree; kept nodes' K and V moved into place

and, between the last two, ``LogitRules.encode`` of sampling.py.  No counterpart
in the reference, which decodes one token at a time.  Everything stays on the
device, so a step can be captured in a CUDA graph.
"""
from __future__ import annotations

import torch

from ._lib import Context, TFError, TF_ERR_INVALID_ARG, lib, on_device
from .paged import PagedKV, PagedKVLayers, _heads, _int32, _stream

_I32 = torch.int32


class DraftTree:
    """Positions and ancestors of drafted trees (tf_draft_tree_plan)."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())
        self.call = lib().tf_draft_tree_plan

    def encode_plan(self, parents, seq_lens, token_starts, positions, ancestors, max_query: int,
                    position_base: int = 0, stream=None):
        """parents [T]: of each node of a request the index of its parent among them, -1 for a root.
        Writes positions [T] (position_base + history + depth) and ancestors [T][words], a bit for every
        node on the way from the root, the node's own among them; rows of no request get -1 and 0."""
        T, B = parents.numel(), seq_lens.numel()
        _int32("DraftTree.encode_plan", parents, seq_lens, token_starts, positions, ancestors)
        if positions.numel() != T or ancestors.dim() != 2 or ancestors.shape[0] != T or token_starts.numel() != B + 1:
            raise TFError(TF_ERR_INVALID_ARG, "DraftTree.encode_plan: sizes of the tensors do not agree")
        on_device("DraftTree.encode_plan", self.ctx.device, parents, seq_lens, token_starts, positions, ancestors)
        st = self.call(self.ctx.handle, parents.data_ptr(), seq_lens.data_ptr(), token_starts.data_ptr(), B, max_query,
                       T, position_base, positions.data_ptr(), ancestors.data_ptr(), ancestors.shape[1],
                       _stream(stream, self.ctx.device))
        if st:
            self.ctx.check(st, "DraftTree.encode_plan")


class TreeAttention:
    """Attention of drafted trees behind a shared prefix (tf_tree_attention)."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())
        self.call = lib().tf_tree_attention

    def workspace_bytes(self, kv: PagedKV, num_q_heads: int, tokens: int, num_requests: int, prefix_len: int,
                        max_query: int) -> int:
        """Enough for every call with at most these sizes."""
        return int(lib().tf_tree_attention_workspace_bytes(self.ctx.handle, kv.ref, num_q_heads, tokens, num_requests,
                                                           prefix_len, max_query))

    def encode(self, q, kv: PagedKV, page_table, seq_lens, token_starts, ancestors, out, workspace, prefix_pages=None,
               prefix_len: int = 0, max_query: int = 1, scale: float | None = None, window: int = 0, positions=None,
               lse=None, stream=None):
        """q, out [T][heads][dim]: request b's nodes, its last positions, are tokens token_starts[b] ..
        token_starts[b+1]; node t sees the history before them (with a window: what is less than `window`
        before positions[t]) and the nodes whose bits are set in ancestors[t].  max_query: the most nodes of
        a request, up to 256.  `lse` (optional): float32 [T][heads].  scale None: dim ** -0.5."""
        T, nq, hd = q.shape
        B = seq_lens.numel()
        if q.dtype != kv.dtype or out.dtype != kv.dtype or out.shape != q.shape or hd != kv.head_dim:
            raise TFError(TF_ERR_INVALID_ARG, "TreeAttention.encode: q, out and the cache do not agree")
        _int32("TreeAttention.encode", page_table, seq_lens, token_starts, ancestors)
        if (page_table.dim() != 2 or page_table.shape[0] != B or token_starts.numel() != B + 1 or ancestors.dim() != 2
                or ancestors.shape[0] != T):
            raise TFError(TF_ERR_INVALID_ARG, "TreeAttention.encode: sizes of the tensors do not agree")
        if prefix_len:
            if prefix_pages is None or prefix_pages.numel() * kv.page_size < prefix_len:
                raise TFError(TF_ERR_INVALID_ARG, "TreeAttention.encode: too few prefix pages")
            _int32("TreeAttention.encode", prefix_pages)
        if positions is not None:
            _int32("TreeAttention.encode", positions)
            if positions.numel() != T:
                raise TFError(TF_ERR_INVALID_ARG, "TreeAttention.encode: a position for every token")
        if lse is not None and (lse.dtype != torch.float32 or lse.numel() != T * nq or not lse.is_contiguous()):
            raise TFError(TF_ERR_INVALID_ARG, "TreeAttention.encode: lse must be contiguous float32 [T][heads]")
        on_device("TreeAttention.encode", self.ctx.device, q, kv.k, kv.v, page_table, seq_lens, token_starts, ancestors,
                  out, workspace, prefix_pages, positions, lse)
        st = self.call(
            self.ctx.handle, q.data_ptr(), _heads(q, "q"), kv.ref, prefix_pages.data_ptr() if prefix_len else None,
            prefix_len, page_table.data_ptr(), page_table.shape[1], seq_lens.data_ptr(), token_starts.data_ptr(), B,
            ancestors.data_ptr(), ancestors.shape[1], None if positions is None else positions.data_ptr(), max_query, T,
            nq, hd ** -0.5 if scale is None else scale, window, out.data_ptr(), _heads(out, "out"),
            None if lse is None else lse.data_ptr(), workspace.data_ptr(), workspace.nbytes,
            _stream(stream, self.ctx.device))
        if st:
            self.ctx.check(st, "TreeAttention.encode")


class DraftAccept:
    """The way down each drafted tree that the model chose, and its K and V put in place
    (tf_draft_accept)."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())
        self.call = lib().tf_draft_accept

    def encode(self, token_ids, parents, choices, seq_lens, token_starts, counts, paths, tokens, targets,
               max_query: int, given=None, layers: PagedKVLayers | None = None, page_table=None, stream=None):
        """token_ids, parents, choices [T]: the nodes, and the token chosen after each.  given (optional):
        how many leading nodes of each request are known tokens, kept without a look (1: the root).  Writes
        counts, targets [requests] and paths, tokens [requests][max_query]: how many nodes are kept and
        which, the new tokens, and the lengths for KVPages.  `layers`: the pools in which the kept nodes'
        K and V move to the positions behind the history (page_table: the requests' pages)."""
        what = "DraftAccept.encode"
        T, B = token_ids.numel(), seq_lens.numel()
        _int32(what, token_ids, parents, choices, seq_lens, token_starts, counts, paths, tokens, targets)
        if (parents.numel() != T or choices.numel() != T or token_starts.numel() != B + 1 or counts.numel() != B
                or targets.numel() != B or paths.numel() != B * max_query or tokens.numel() != B * max_query):
            raise TFError(TF_ERR_INVALID_ARG, f"{what}: sizes of the tensors do not agree")
        if given is not None:
            _int32(what, given)
            if given.numel() != B:
                raise TFError(TF_ERR_INVALID_ARG, f"{what}: given is one number a request")
        on_device(what, self.ctx.device, token_ids, parents, choices, seq_lens, token_starts, counts, paths, tokens,
                  targets, given)
        n = 0 if layers is None else layers.layers
        if n:
            if page_table is None or page_table.dim() != 2 or page_table.shape[0] != B:
                raise TFError(TF_ERR_INVALID_ARG, f"{what}: pools need the requests' page table")
            _int32(what, page_table)
            on_device(what, self.ctx.device, layers.k, layers.v, page_table)
        st = self.call(self.ctx.handle, token_ids.data_ptr(), parents.data_ptr(), choices.data_ptr(),
                       None if given is None else given.data_ptr(), seq_lens.data_ptr(), token_starts.data_ptr(), B,
                       max_query, T, counts.data_ptr(), paths.data_ptr(), tokens.data_ptr(), targets.data_ptr(),
                       layers.ref if n else None, layers.layer_stride if n else 0, n,
                       page_table.data_ptr() if n else None, page_table.shape[1] if n else 0,
                       _stream(stream, self.ctx.device))
        if st:
            self.ctx.check(st, what)
