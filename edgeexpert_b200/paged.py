"""Serving a ragged batch: a paged KV cache whose requests have different
lengths and share one long prefix.

* ``KVPages.encode_resize``          request lengths -> page tables, slots, positions (on the device)
* ``RotaryKVWrite.encode``           head norms + rotary positions; K and V into the tokens' slots
* ``SharedPrefixAttention.encode``   attention over the shared prefix and each request's own pages
* ``PagedKVCache``, ``PagedDecoder``  the decoder of decoder.py on such a batch, with the three operators

The operators have no counterpart in the reference, which decodes one sequence
from a contiguous cache.  Lengths, tables, slots and positions are int32 CUDA
tensors; nothing is read back, so a step can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import Context, PagedKVDesc, TFError, TF_ERR_INVALID_ARG, TF_OK, lib, raw_stream as _stream, status_string
from .decoder import Decoder

_I32 = torch.int32
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_LAYOUTS = {"half": 0, "interleaved": 1}
_MAX_STEP = 256  # rows that tf_lm_head_greedy takes
_SCALINGS = {None: 0, "linear": 1, "base": 2, "ramp": 3, "bands": 4}


def _heads(t, what: str) -> int:
    """Token stride of a [tokens][heads][dim] tensor whose heads lie side by side."""
    if t.is_contiguous() and t.dim() == 3:
        return t.shape[1] * t.shape[2]
    if t.dim() != 3 or t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != t.shape[2]):
        raise TFError(TF_ERR_INVALID_ARG, f"{what} must be [tokens][heads][dim] with contiguous heads")
    return t.stride(0)


def _int32(what: str, *tensors):
    for t in tensors:
        if t.dtype is not _I32 or not t.is_contiguous():
            raise TFError(TF_ERR_INVALID_ARG, f"{what}: lengths, tables, slots and positions are contiguous int32 tensors")


class PagedKV:
    """One layer's K and V pools, [page][position][head][dim] tensors of one
    dtype (fp16 or bf16) and of any strides with dim innermost: a
    [page][head][position][dim] pool is passed as its transposed view."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.stride(3) != 1:
            raise TFError(TF_ERR_INVALID_ARG, "k and v must be alike: [page][position][head][dim], dim innermost")
        if k.dtype not in _DTYPES:
            raise TFError(TF_ERR_INVALID_ARG, f"cache dtype {k.dtype}: float16 or bfloat16")
        self.k, self.v, self.dtype = k, v, k.dtype
        self.num_pages, self.page_size, self.num_kv_heads, self.head_dim = k.shape
        self.desc = PagedKVDesc(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), self.num_pages,
                                self.page_size, self.num_kv_heads, self.head_dim, _DTYPES[k.dtype])
        self.ref = C.byref(self.desc)


class PagedKVLayers:
    """The pools of all layers, [layer][page][position][head][dim]: `layer[i]` is layer i's PagedKV."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 5 or k.shape != v.shape or k.stride() != v.stride():
            raise TFError(TF_ERR_INVALID_ARG, "k and v must be alike: [layer][page][position][head][dim]")
        self.layer = [PagedKV(k[i], v[i]) for i in range(k.shape[0])]
        self.layers, self.layer_stride = k.shape[0], k.stride(0)
        self.k, self.v, self.ref = k, v, self.layer[0].ref if self.layer else None


class KVPages:
    """The page tables of a ragged batch (tf_kv_pages_resize)."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())
        self.call = lib().tf_kv_pages_resize

    @staticmethod
    def workspace_bytes(num_requests: int) -> int:
        return int(lib().tf_kv_pages_workspace_bytes(num_requests))

    def encode_resize(self, seq_lens, targets, page_table, free_ring, free_state, seq_lens_out, free_state_out,
                      token_starts, slots, positions, requests, page_size: int, workspace, position_base: int = 0,
                      stream=None):
        """Grow or shrink every request to its target length: pages move between
        `free_ring` and `page_table` [requests][max_pages], and every token added
        gets its slot, position and request (-1 beyond the last).  seq_lens_out /
        free_state_out may be seq_lens / free_state.  free_state = {head, count,
        requests refused, tokens added}."""
        B, max_tokens = seq_lens.numel(), slots.numel()
        _int32("KVPages.encode_resize", seq_lens, targets, page_table, free_ring, free_state, seq_lens_out,
               free_state_out, token_starts, slots, positions, requests)
        if (targets.numel() != B or seq_lens_out.numel() != B or token_starts.numel() != B + 1
                or page_table.dim() != 2 or page_table.shape[0] != B or free_state.numel() != 4
                or free_state_out.numel() != 4 or positions.numel() != max_tokens or requests.numel() != max_tokens):
            raise TFError(TF_ERR_INVALID_ARG, "KVPages.encode_resize: sizes of the tensors do not agree")
        st = self.call(
            self.ctx.handle, seq_lens.data_ptr(), targets.data_ptr(), B, page_table.data_ptr(), page_table.shape[1],
            free_ring.data_ptr(), free_ring.numel(), free_state.data_ptr(), page_size, position_base,
            seq_lens_out.data_ptr(), free_state_out.data_ptr(), token_starts.data_ptr(), slots.data_ptr(),
            positions.data_ptr(), requests.data_ptr(), max_tokens, workspace.data_ptr(),
            workspace.nbytes, _stream(stream, self.ctx.device))
        if st:
            self.ctx.check(st, "KVPages.encode_resize")


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                     original_context: float = 0.0, low: float = 1.0, high: float = 32.0, device="cuda"):
    """(radians per position of each pair as a float64 tensor, attention factor)
    for RotaryKVWrite.  scaling: None, "linear", "base", "ramp" (low / high =
    turns over the original context below which a pair is slowed fully and
    above which it is kept) or "bands" (the same, linear in the turns)."""
    if scaling not in _SCALINGS:
        raise TFError(TF_ERR_INVALID_ARG, f"rope_frequencies: unknown scaling {scaling!r}")
    out, mul = (C.c_double * max(1, rotary_dim // 2))(), C.c_double(1.0)
    st = lib().tf_rope_frequencies(rotary_dim, theta, _SCALINGS[scaling], factor, original_context, low, high, out,
                                   C.byref(mul))
    if st != TF_OK:
        raise TFError(st, f"rope_frequencies: {status_string(st)}")
    return torch.tensor(list(out)[:rotary_dim // 2], dtype=torch.float64, device=device), mul.value


class RotaryKVWrite:
    """Per-head norms, rotary positions and the write into the paged cache
    (tf_rope_kv_write)."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())
        self.call = lib().tf_rope_kv_write

    def encode(self, q, k, v, q_out, kv: PagedKV, slots, positions, inv_freq, rotary_dim: int | None = None,
               layout: str = "half", attention_factor: float = 1.0, q_weight=None, k_weight=None, norm: bool = False,
               eps: float = 1e-6, stream=None):
        """q, q_out [T][heads][dim], k, v [T][kv heads][dim] (views of a fused
        projection are fine); q_out may be q."""
        T, nq, hd = q.shape
        rot = hd if rotary_dim is None else rotary_dim
        dtype = kv.dtype
        if layout not in _LAYOUTS:
            raise TFError(TF_ERR_INVALID_ARG, f"RotaryKVWrite.encode: unknown layout {layout!r}")
        if q.dtype is not dtype or k.dtype is not dtype or v.dtype is not dtype or q_out.dtype is not dtype:
            raise TFError(TF_ERR_INVALID_ARG, "RotaryKVWrite.encode: q, k, v, q_out and the cache must have one dtype")
        shape = k.shape
        if shape != v.shape or shape != (T, kv.num_kv_heads, kv.head_dim) or q_out.shape != q.shape or hd != kv.head_dim:
            raise TFError(TF_ERR_INVALID_ARG, "RotaryKVWrite.encode: shapes of q, k, v and the cache do not agree")
        _int32("RotaryKVWrite.encode", slots, positions)
        if (slots.numel() != T or positions.numel() != T or inv_freq.dtype is not torch.float64
                or inv_freq.numel() * 2 != rot or not inv_freq.is_contiguous()):
            raise TFError(TF_ERR_INVALID_ARG,
                          "RotaryKVWrite.encode: a slot and position per token, a contiguous float64 per pair")
        if q_weight is not None or k_weight is not None:
            for w in (q_weight, k_weight):
                if w is not None and (w.dtype is not torch.bfloat16 or w.numel() != hd or not w.is_contiguous()):
                    raise TFError(TF_ERR_INVALID_ARG, "RotaryKVWrite.encode: norm weights are contiguous bf16 [head_dim]")
        st = self.call(
            self.ctx.handle, q.data_ptr(), _heads(q, "q"), k.data_ptr(), _heads(k, "k"), v.data_ptr(), _heads(v, "v"),
            q_out.data_ptr(), _heads(q_out, "q_out"), kv.ref, slots.data_ptr(), positions.data_ptr(),
            inv_freq.data_ptr(), rot, _LAYOUTS[layout], attention_factor, int(norm),
            None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
            T, nq, _stream(stream, self.ctx.device))
        if st:
            self.ctx.check(st, "RotaryKVWrite.encode")


class SharedPrefixAttention:
    """Causal attention of a ragged batch behind a shared prefix
    (tf_shared_prefix_attention)."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())
        self.call = lib().tf_shared_prefix_attention

    def workspace_bytes(self, kv: PagedKV, num_q_heads: int, tokens: int, num_requests: int, prefix_len: int,
                        max_query: int) -> int:
        """Enough for every call with at most these sizes."""
        return int(lib().tf_shared_prefix_attention_workspace_bytes(self.ctx.handle, kv.ref, num_q_heads, tokens,
                                                                    num_requests, prefix_len, max_query))

    def encode(self, q, kv: PagedKV, page_table, seq_lens, token_starts, out, workspace, prefix_pages=None,
               prefix_len: int = 0, max_query: int = 1, scale: float | None = None, window: int = 0, lse=None,
               stream=None):
        """q, out [T][heads][dim]: request b's last positions are tokens
        token_starts[b] .. token_starts[b+1].  `lse` (optional): float32
        [T][heads].  scale None: dim ** -0.5."""
        T, nq, hd = q.shape
        B = seq_lens.numel()
        if q.dtype != kv.dtype or out.dtype != kv.dtype or out.shape != q.shape or hd != kv.head_dim:
            raise TFError(TF_ERR_INVALID_ARG, "SharedPrefixAttention.encode: q, out and the cache do not agree")
        _int32("SharedPrefixAttention.encode", page_table, seq_lens, token_starts)
        if page_table.dim() != 2 or page_table.shape[0] != B or token_starts.numel() != B + 1:
            raise TFError(TF_ERR_INVALID_ARG, "SharedPrefixAttention.encode: sizes of the tensors do not agree")
        if prefix_len:
            if prefix_pages is None or prefix_pages.numel() * kv.page_size < prefix_len:
                raise TFError(TF_ERR_INVALID_ARG, "SharedPrefixAttention.encode: too few prefix pages")
            _int32("SharedPrefixAttention.encode", prefix_pages)
        if lse is not None and (lse.dtype != torch.float32 or lse.numel() != T * nq or not lse.is_contiguous()):
            raise TFError(TF_ERR_INVALID_ARG, "SharedPrefixAttention.encode: lse must be contiguous float32 [T][heads]")
        st = self.call(
            self.ctx.handle, q.data_ptr(), _heads(q, "q"), kv.ref, prefix_pages.data_ptr() if prefix_len else None,
            prefix_len, page_table.data_ptr(), page_table.shape[1], seq_lens.data_ptr(), token_starts.data_ptr(), B,
            max_query, T, nq, hd ** -0.5 if scale is None else scale, window, out.data_ptr(), _heads(out, "out"),
            None if lse is None else lse.data_ptr(), workspace.data_ptr(), workspace.nbytes,
            _stream(stream, self.ctx.device))
        if st:
            self.ctx.check(st, "SharedPrefixAttention.encode")


class PagedKVCache:
    """The pools of every layer, and one set of page tables for all of them: a
    request's position has the same slot in each layer.  The page tables live on
    the device; `resize` is the only thing that changes them."""

    def __init__(self, layers: int, num_kv_heads: int, head_dim: int, num_requests: int, num_pages: int,
                 max_pages: int, max_tokens: int, page_size: int = 16, dtype=torch.float16, device="cuda",
                 context: Context | None = None):
        """num_pages: of each layer's pool; max_pages: of one request; max_tokens: added in one step."""
        def i32(*shape, fill=0):
            return torch.full(shape, fill, dtype=_I32, device=device)

        shape = (layers, num_pages, page_size, num_kv_heads, head_dim)
        self.k, self.v = torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)
        self.layers = PagedKVLayers(self.k, self.v)
        self.layer = self.layers.layer
        self.page_size, self.num_requests, self.max_tokens = page_size, num_requests, max_tokens
        self.seq_lens, self.page_table = i32(num_requests), i32(num_requests, max_pages, fill=-1)
        self.free_ring = torch.arange(num_pages, dtype=_I32, device=device)
        self.free_state = torch.tensor([0, num_pages, 0, 0], dtype=_I32, device=device)
        self.token_starts = i32(num_requests + 1)
        self.slots, self.positions, self.requests = (i32(max_tokens, fill=-1) for _ in range(3))
        self.prefix_pages, self.prefix_len = None, 0
        self.pages = KVPages(context)
        self.workspace = torch.empty(KVPages.workspace_bytes(num_requests), dtype=torch.uint8, device=device)

    def resize(self, targets, stream=None):
        """Bring the requests to `targets` positions of their own (int32, on the device; -1 leaves one
        alone, 0 frees its pages).  free_state then holds {head, free pages, requests refused, tokens added}."""
        self.pages.encode_resize(self.seq_lens, targets, self.page_table, self.free_ring, self.free_state,
                                 self.seq_lens, self.free_state, self.token_starts, self.slots, self.positions,
                                 self.requests, self.page_size, self.workspace, position_base=self.prefix_len,
                                 stream=stream)

    def share(self, request: int, length: int, stream=None):
        """Make the `length` positions that `request` holds, all of them, the prefix of all requests:
        its pages leave the tables and stay out of the free ring for as long as the cache lives.
        The others must be empty.  Reads the lengths back (once in the cache's life)."""
        if self.prefix_len:
            raise TFError(TF_ERR_INVALID_ARG, "PagedKVCache.share: there is a prefix already")
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, self.seq_lens.device)
        with torch.cuda.stream(stream):  # (None: the current one)
            held = self.seq_lens.tolist()
            if length <= 0 or held != [length if b == request else 0 for b in range(self.num_requests)]:
                raise TFError(TF_ERR_INVALID_ARG, f"PagedKVCache.share: the requests hold {held} positions; "
                              f"request {request} must hold {length} and the others none")
            self.prefix_pages = self.page_table[request, :-(-length // self.page_size)].clone()
            self.seq_lens[request] = 0
        self.prefix_len = length


class PagedDecoder(Decoder):
    """The decoder on a ragged batch: a step adds any number of tokens to each
    request (a prompt, a draft, one token, none), up to T in all, and gives the
    next token after every one of them.  Rows beyond the tokens added are padding."""

    def __init__(self, weights, T: int, cache: PagedKVCache, max_query: int = 1, context: Context | None = None,
                 device=None):
        """T: the most tokens of a step, up to 256 (the rows of the LM head).  max_query: the most
        that a step adds to one request."""
        if not 0 < T <= _MAX_STEP:
            raise TFError(TF_ERR_INVALID_ARG, f"PagedDecoder: a step has 1 to {_MAX_STEP} tokens")
        super().__init__(weights, T, _NoContiguousCache(), context, device)
        cfg = weights.cfg
        if cache.max_tokens != T:
            raise TFError(TF_ERR_INVALID_ARG, "PagedDecoder: the cache must take as many tokens a step")
        self.kv, self.max_query = cache, max_query
        dev = self.q.device
        self.k_rows, self.v_rows = (torch.empty(T, cfg.num_kv_heads * cfg.head_dim, dtype=torch.float16, device=dev)
                                    for _ in range(2))
        self.inv_freq, self.rope_factor = rope_frequencies(cfg.head_dim, cfg.rope_theta, device=dev)
        self.rope, self.attention = RotaryKVWrite(self.ctx), SharedPrefixAttention(self.ctx)
        self.workspace, self._workspaces = None, []
        self.ids = torch.zeros(T, dtype=_I32, device=dev)  # the tokens of a step's rows

    def _attend(self, i: int, position, stream):
        cfg, L, T, kv = self.cfg, self.w.layers[i], self.T, self.kv
        hd, nq, nkv = cfg.head_dim, cfg.num_q_heads, cfg.num_kv_heads
        self._proj(L.q, self.normed, self.q, stream)
        self._proj(L.k, self.normed, self.k_rows, stream)
        self._proj(L.v, self.normed, self.v_rows, stream)
        q = self.q.view(T, nq, hd)
        self.rope.encode(q, self.k_rows.view(T, nkv, hd), self.v_rows.view(T, nkv, hd), q, kv.layer[i], kv.slots,
                         self._row_positions(), self.inv_freq, attention_factor=self.rope_factor, q_weight=L.q_norm,
                         k_weight=L.k_norm, norm=True, eps=cfg.eps, stream=stream)
        self._attend_rows(q, i, self.attn.view(T, nq, hd), stream)

    def _row_positions(self):
        return self.kv.positions

    def _attend_rows(self, q, i: int, out, stream):
        kv = self.kv
        self.attention.encode(q, kv.layer[i], kv.page_table, kv.seq_lens, kv.token_starts, out, self.workspace,
                              prefix_pages=kv.prefix_pages, prefix_len=kv.prefix_len, max_query=self.max_query, scale=1.0,
                              stream=stream)

    def _workspace_bytes(self) -> int:
        kv = self.kv
        return self.attention.workspace_bytes(kv.layer[0], self.cfg.num_q_heads, self.T, kv.num_requests, kv.prefix_len,
                                              self.max_query)

    def _resize(self, token_ids, targets, stream):
        """The page tables brought to `targets`, and self.ids = the tokens of the requests that
        were granted.  The list holds the tokens of all that asked, the rows those of the granted
        ones alone; a request whose tokens the list does not hold to the end is refused.  Returns
        every row's place in the list (0 for padding, None for an empty list)."""
        kv, n = self.kv, token_ids.numel()
        before = kv.seq_lens.clone()
        asked = torch.maximum(targets, before) - before
        ends = asked.cumsum(0)  # of the requests' tokens in the list
        kv.resize(torch.where((ends > n) & (asked > 0), 2 ** 31 - 1, targets), stream)
        first = ends - asked - before - kv.prefix_len  # + a token's position = its place in the list
        if n == 0:
            self.ids.zero_()
            return None
        at = (first[kv.requests.clamp(min=0)] + kv.positions).clamp_(0, n - 1)
        torch.mul(token_ids[at], kv.requests >= 0, out=self.ids)
        return at

    def step(self, token_ids, targets, stream=None):
        """token_ids (up to T): the tokens to add, request after request, of every request that
        is to grow; targets: every request's length with them.  Both int32, on the device.  A
        request that can't have its pages is refused and keeps its length (what it asked for
        counts before later requests' pages all the same); the others get their own tokens.  Next
        tokens in self.tokens, row by row of the tokens added: row i is position kv.positions[i]
        of request kv.requests[i], and kv.free_state tells how many requests were refused."""
        self._check_step("PagedDecoder.step", token_ids, targets)
        with torch.cuda.stream(stream):  # (None: the current one)
            self._make_workspace()
            self._resize(token_ids, targets, stream)
        return self._run_rows(stream)

    def _check_step(self, name: str, token_ids, targets, **more):
        for what, t in dict(token_ids=token_ids, targets=targets, **more).items():
            if t.dtype is not _I32 or t.dim() != 1 or t.device != self.ids.device:
                raise TFError(TF_ERR_INVALID_ARG, f"{name}: {what} must be a vector of int32 on {self.ids.device}")
        if token_ids.numel() > self.T or targets.numel() != self.kv.num_requests:
            raise TFError(TF_ERR_INVALID_ARG, f"{name}: up to T tokens, a target per request")

    def _make_workspace(self):
        self.workspace = self._larger(self.workspace, self._workspace_bytes())

    def _larger(self, workspace, need: int):
        """`workspace`, or one of `need` bytes in its place.  The old one stays: a step that was captured
        in a graph goes on writing there.  Each is at least twice the one before, so that all of them
        together are at most twice the last, however slowly the need grows."""
        if workspace is not None:
            if workspace.nbytes >= need:
                return workspace
            need = max(need, 2 * workspace.nbytes)
        self._workspaces.append(torch.empty(need, dtype=torch.uint8, device=self.q.device))
        return self._workspaces[-1]

    def _run_rows(self, stream):
        self.launches = 0
        self.embed(self.ids, stream)
        for i in range(self.cfg.layers):
            self.layer(i, None, stream)
        self.lm_head(stream)
        return self.tokens


class _NoContiguousCache:
    ctx_len = 1  # Decoder sizes its own attention's scratch by it
