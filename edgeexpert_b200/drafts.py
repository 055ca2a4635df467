"""Drafted trees in a ragged batch on a paged KV cache: a step checks many guessed
tokens of each request at once and keeps the way that the model itself chose.

* ``DraftTree.encode_plan``    parents -> positions and ancestors of every node
* ``TreeAttention.encode``     attention of the nodes over prefix, history and ancestors
* ``DraftAccept.encode``       the walk down each tree; kept nodes' K and V moved into place

and, between the last two, ``LogitRules.encode`` of sampling.py; ``DraftDecoder``
is the decoder of paged.py with all four.  No counterpart in the reference, which
decodes one token at a time.  Everything stays on the device, so a step can be
captured in a CUDA graph.
"""
from __future__ import annotations

import torch

from ._lib import Context, TFError, TF_ERR_INVALID_ARG, int32_on_device, lib, on_device, raw_stream
from .paged import PagedDecoder, PagedKV, PagedKVCache, PagedKVLayers, _heads
from .sampling import LogitRules


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
        device = self.ctx.device
        int32_on_device("DraftTree.encode_plan", device, parents, seq_lens, token_starts, positions, ancestors)
        if positions.numel() != T or ancestors.dim() != 2 or ancestors.shape[0] != T or token_starts.numel() != B + 1:
            raise TFError(TF_ERR_INVALID_ARG, "DraftTree.encode_plan: sizes of the tensors do not agree")
        st = self.call(self.ctx.handle, parents.data_ptr(), seq_lens.data_ptr(), token_starts.data_ptr(), B, max_query,
                       T, position_base, positions.data_ptr(), ancestors.data_ptr(), ancestors.shape[1],
                       raw_stream(stream, device))
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
        what, device = "TreeAttention.encode", self.ctx.device
        int32_on_device(what, device, page_table, seq_lens, token_starts, ancestors)
        if (page_table.dim() != 2 or page_table.shape[0] != B or token_starts.numel() != B + 1 or ancestors.dim() != 2
                or ancestors.shape[0] != T):
            raise TFError(TF_ERR_INVALID_ARG, "TreeAttention.encode: sizes of the tensors do not agree")
        if prefix_len:
            if prefix_pages is None or prefix_pages.numel() * kv.page_size < prefix_len:
                raise TFError(TF_ERR_INVALID_ARG, "TreeAttention.encode: too few prefix pages")
            int32_on_device(what, device, prefix_pages)
        if positions is not None:
            int32_on_device(what, device, positions)
            if positions.numel() != T:
                raise TFError(TF_ERR_INVALID_ARG, "TreeAttention.encode: a position for every token")
        if lse is not None and (lse.dtype != torch.float32 or lse.numel() != T * nq or not lse.is_contiguous()):
            raise TFError(TF_ERR_INVALID_ARG, "TreeAttention.encode: lse must be contiguous float32 [T][heads]")
        on_device(what, device, q, kv.k, kv.v, out, workspace, lse)
        st = self.call(
            self.ctx.handle, q.data_ptr(), _heads(q, "q"), kv.ref, prefix_pages.data_ptr() if prefix_len else None,
            prefix_len, page_table.data_ptr(), page_table.shape[1], seq_lens.data_ptr(), token_starts.data_ptr(), B,
            ancestors.data_ptr(), ancestors.shape[1], None if positions is None else positions.data_ptr(), max_query, T,
            nq, hd ** -0.5 if scale is None else scale, window, out.data_ptr(), _heads(out, "out"),
            None if lse is None else lse.data_ptr(), workspace.data_ptr(), workspace.nbytes,
            raw_stream(stream, device))
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
        what, device = "DraftAccept.encode", self.ctx.device
        T, B = token_ids.numel(), seq_lens.numel()
        int32_on_device(what, device, token_ids, parents, choices, seq_lens, token_starts, counts, paths, tokens, targets)
        if (parents.numel() != T or choices.numel() != T or token_starts.numel() != B + 1 or counts.numel() != B
                or targets.numel() != B or paths.numel() != B * max_query or tokens.numel() != B * max_query):
            raise TFError(TF_ERR_INVALID_ARG, f"{what}: sizes of the tensors do not agree")
        if given is not None:
            int32_on_device(what, device, given)
            if given.numel() != B:
                raise TFError(TF_ERR_INVALID_ARG, f"{what}: given is one number a request")
        n = 0 if layers is None else layers.layers
        if n:
            if page_table is None or page_table.dim() != 2 or page_table.shape[0] != B:
                raise TFError(TF_ERR_INVALID_ARG, f"{what}: pools need the requests' page table")
            int32_on_device(what, device, page_table)
            on_device(what, device, layers.k, layers.v)
        st = self.call(self.ctx.handle, token_ids.data_ptr(), parents.data_ptr(), choices.data_ptr(),
                       None if given is None else given.data_ptr(), seq_lens.data_ptr(), token_starts.data_ptr(), B,
                       max_query, T, counts.data_ptr(), paths.data_ptr(), tokens.data_ptr(), targets.data_ptr(),
                       layers.ref if n else None, layers.layer_stride if n else 0, n,
                       page_table.data_ptr() if n else None, page_table.shape[1] if n else 0,
                       raw_stream(stream, device))
        if st:
            self.ctx.check(st, what)


class DraftDecoder(PagedDecoder):
    """PagedDecoder with steps that check drafted trees: `draft` adds the nodes of each request's tree,
    chooses a token after every one, keeps the way that the choices take from the root, and gives the
    pages of the others back.  `step` is as before."""

    def __init__(self, weights, T: int, cache: PagedKVCache, max_query: int = 1, context: Context | None = None,
                 device=None):
        super().__init__(weights, T, cache, max_query, context, device)
        if max_query > 256:
            raise TFError(TF_ERR_INVALID_ARG, "DraftDecoder: a tree has up to 256 nodes")
        dev, B = self.q.device, cache.num_requests

        def i32(*shape):
            return torch.zeros(shape, dtype=torch.int32, device=dev)

        self.tree, self.tree_attention = DraftTree(self.ctx), TreeAttention(self.ctx)
        self.rules, self.accept = LogitRules(self.ctx), DraftAccept(self.ctx)
        self.rules_checks = LogitRules(self.ctx)
        self.rules_checks.call = lambda *args: 0  # the rules' checks alone, before a step changes anything
        self.parents, self.node_positions, self.ancestors = i32(T), i32(T), i32(T, -(-max_query // 32))
        self.counts, self.targets = i32(B), i32(B)
        self.paths, self.new_tokens = i32(B, max_query), i32(B, max_query)
        self.draft_starts, self.draft_state, self.mask_rows = i32(B + 1), i32(4), i32(T)
        self.rules_workspace = None
        self._drafting = False

    def _row_positions(self):
        return self.node_positions if self._drafting else super()._row_positions()

    def _attend_rows(self, q, i: int, out, stream):
        if not self._drafting:
            return super()._attend_rows(q, i, out, stream)
        kv = self.kv
        self.tree_attention.encode(q, kv.layer[i], kv.page_table, kv.seq_lens, kv.token_starts, self.ancestors, out,
                                   self.workspace, prefix_pages=kv.prefix_pages, prefix_len=kv.prefix_len,
                                   max_query=self.max_query, scale=1.0, stream=stream)

    def _workspace_bytes(self) -> int:
        kv = self.kv
        return max(super()._workspace_bytes(), self.tree_attention.workspace_bytes(
            kv.layer[0], self.cfg.num_q_heads, self.T, kv.num_requests, kv.prefix_len, self.max_query))

    def draft(self, token_ids, parents, targets, given=None, rules: dict | None = None, stream=None):
        """token_ids, targets: as in step, the tokens of a request being the nodes of its tree (up to
        max_query).  parents: of each token the index of its parent among its request's, below its own,
        or -1 for the root (the first).  given (optional): how many leading tokens of each request are
        known and kept without a look, a prompt's for instance; 1, the root, without it.  rules: what
        LogitRules.encode takes for the requests (history, repetition, biases, allowed ...); allowed_rows is
        of each token of the list the row of `allowed` that holds for the choice after it, -1: none (without
        allowed_rows token t's row is t), whichever requests are refused.  The tokens, the root's too, count
        as said on their way down, so that `history` ends before the root; those of a request whose given is
        above 1 count as its prompt (prompt_nodes says otherwise: of each request how many of its first
        tokens are the prompt's, 1 for a prompt of one token, 0 for known tokens of the output).  self.logits
        then holds the logits under the rules, self.tokens the choice after every node.

        Returns (counts, new_tokens), on the device and the decoder's own, for the next step writes there
        again: how many nodes of each request are kept, and
        [requests][max_query] the counts - given + 1 tokens that are new, -1 behind them.  The last of
        them is not in the cache yet: it is the next root.  self.paths: which nodes are kept.  The cache
        then holds the kept nodes alone; rows i of this step were tokens draft_starts[b] .. of request b,
        and draft_state is what free_state was after they were added."""
        kv = self.kv
        more = {} if given is None else dict(given=given)
        self._check_step("DraftDecoder.draft", token_ids, targets, parents=parents, **more)
        if parents.numel() != token_ids.numel() or (given is not None and given.numel() != kv.num_requests):
            raise TFError(TF_ERR_INVALID_ARG, "DraftDecoder.draft: a parent for every token, given for every request")
        allowed, rows = (None, None) if rules is None else (rules.get("allowed"), rules.get("allowed_rows"))
        if rows is not None:
            self._check_step("DraftDecoder.draft", token_ids, targets, allowed_rows=rows)
        if (allowed if rows is None else rows) is not None and len(allowed if rows is None else rows) < len(token_ids):
            raise TFError(TF_ERR_INVALID_ARG, "DraftDecoder.draft: a row of allowed tokens for every token")
        with torch.cuda.stream(stream):  # (None: the current one)
            self._make_workspace()
            if rules is not None:
                if allowed is not None:
                    rules = {**rules, "allowed_rows": self.mask_rows}
                if given is not None and rules.get("prompt_nodes") is None:
                    rules = {**rules, "prompt_nodes": torch.where(given > 1, given, 0)}
                self._make_rules_workspace(rules)
                self._apply(self.rules_checks, rules, stream)
            at = self._resize(token_ids, targets, stream)
            if at is None:
                self.parents.fill_(-1)
            else:
                self.parents.copy_(torch.where(kv.requests >= 0, parents[at], -1))
            if allowed is not None:  # from the list's order to the rows of those that were granted
                if at is None:
                    self.mask_rows.fill_(-1)
                else:
                    self.mask_rows.copy_(torch.where(kv.requests >= 0, at if rows is None else rows[at], -1))
            self.draft_starts.copy_(kv.token_starts)
            self.draft_state.copy_(kv.free_state)
        try:
            self._check_nodes(given, rules, stream)
        except Exception:  # what does not fail for the step's arguments, which are checked: no nodes are left
            with torch.cuda.stream(stream):
                kv.resize(kv.seq_lens - (self.draft_starts[1:] - self.draft_starts[:-1]), stream)
            raise
        kv.resize(self.targets, stream)
        return self.counts, self.new_tokens

    def _make_rules_workspace(self, rules):
        history, biases = rules.get("history"), rules.get("bias_tokens")
        need = self.rules.workspace_bytes(self.T, self.cfg.vocab, self.kv.num_requests,
                                          0 if history is None else history.shape[-1],
                                          0 if biases is None else biases.numel())
        if need == 0:
            raise TFError(TF_ERR_INVALID_ARG, f"DraftDecoder.draft: no rules for {self.cfg.vocab} tokens")
        self.rules_workspace = self._larger(self.rules_workspace, need)

    def _apply(self, operator: LogitRules, rules, stream):
        operator.encode(self.logits, self.logits, self.kv.token_starts, self.rules_workspace, max_query=self.max_query,
                        token_ids=self.ids, ancestors=self.ancestors, tokens=self.tokens, stream=stream, **rules)

    def _check_nodes(self, given, rules, stream):
        """The nodes' positions, logits, choices and ways; self.targets: the lengths with the kept ones."""
        kv = self.kv
        self.tree.encode_plan(self.parents, kv.seq_lens, kv.token_starts, self.node_positions, self.ancestors,
                              self.max_query, position_base=kv.prefix_len, stream=stream)
        self._drafting = True
        try:
            self._run_rows(stream)
        finally:
            self._drafting = False
        if rules is not None:
            self._apply(self.rules, rules, stream)
        self.accept.encode(self.ids, self.parents, self.tokens, kv.seq_lens, kv.token_starts, self.counts, self.paths,
                           self.new_tokens, self.targets, self.max_query, given=given, layers=kv.layers,
                           page_table=kv.page_table, stream=stream)
