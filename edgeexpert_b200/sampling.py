"""Output-head sampling, mirroring the reference's LogitSoftcapSoftmax,
Sample and SampleTopK64 encoders (Kernels/Sampling/LogitOutput.swift;
Metal/Sampling/logit.metal:42-617) on libtfcuda.so; and, without a counterpart
there, LogitRules: penalties, biases and grammar masks on the logits of a
ragged batch before any of them."""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import Context, LogitRulesDesc, TF_ERR_INVALID_ARG, TFError, lib, ptr, raw_stream, stream_ptr

_LOGITS = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class LogitSoftcapSoftmax:
    """probs = softmax(softcap * tanh(logits / softcap)), fp16 out (Gemma 4: softcap 30)."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())

    def encode(self, logits, probs, v: int, softcap: float = 30.0, rows: int = 1, stream=None):
        fp32 = 1 if logits.dtype == torch.float32 else 0
        st = lib().tf_softcap_softmax(self.ctx.handle, ptr(logits), fp32, ptr(probs), v, rows, softcap,
                                      stream_ptr(stream))
        self.ctx.check(st, "LogitSoftcapSoftmax.encode")


class Sample:
    """Greedy / temperature / top-k / top-p sampler on fp16 probabilities."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())

    def encode(self, probs, out_token, v: int, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
               seed: int = 0, position: int = 0, stream=None):
        st = lib().tf_sample(self.ctx.handle, ptr(probs), v, temperature, top_k, top_p, seed & 0xFFFFFFFFFFFFFFFF,
                             position, ptr(out_token), stream_ptr(stream))
        self.ctx.check(st, "Sample.encode")


class SampleTopK64:
    """The three-stage top-64 sampler."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())

    def encode(self, probs, out_token, v: int, temperature: float = 1.0, top_p: float = 1.0, seed: int = 0,
               stream=None):
        st = lib().tf_sample_topk64(self.ctx.handle, ptr(probs), v, temperature, top_p, seed & 0xFFFFFFFFFFFFFFFF,
                                    ptr(out_token), stream_ptr(stream))
        self.ctx.check(st, "SampleTopK64.encode")


class LogitRules:
    """Penalties for repeated tokens, biases and grammar masks on the logits of a ragged batch, and the
    best token under them (tf_logit_rules_apply)."""

    def __init__(self, context: Context | None = None):
        self.ctx = context or Context.get(torch.cuda.current_device())
        self.call = lib().tf_logit_rules_apply

    @staticmethod
    def workspace_bytes(rows: int, vocab: int, requests: int, history: int = 0, biases: int = 0) -> int:
        """Enough for every call with at most these sizes (history: the width of `history`, biases: all
        requests' entries)."""
        return int(lib().tf_logit_rules_workspace_bytes(rows, vocab, requests, history, biases))

    def _place(self, t, dtype, n: int, what: str):
        """Where a vector of n values is (None: nowhere)."""
        if t is None:
            return None
        if t.dtype is not dtype or t.numel() != n or not t.is_contiguous():
            raise TFError(TF_ERR_INVALID_ARG, f"LogitRules.encode: {what}: {n} contiguous values of {dtype}")
        return self._here(t, what)

    def _matrix(self, t, rows: int, what: str, least: int | None = None):
        """Where an int32 matrix is, whose rows have all of their values, or the first `least`, to themselves."""
        if t.dtype is not torch.int32 or t.dim() != 2 or (rows >= 0 and t.shape[0] != rows) or (
                t.shape[1] > 1 and t.stride(1) != 1) or (
                t.shape[0] > 1 and t.stride(0) < (t.shape[1] if least is None else least)):
            raise TFError(TF_ERR_INVALID_ARG, f"LogitRules.encode: {what} must be an int32 matrix, rows contiguous")
        return self._here(t, what)

    def _here(self, t, what: str):
        if t.get_device() != self.ctx.device:
            raise TFError(TF_ERR_INVALID_ARG, f"LogitRules.encode: {what} on {t.device}, the context is on "
                          f"cuda:{self.ctx.device}")
        return t.data_ptr()

    def encode(self, logits, out, token_starts, workspace, max_query: int = 1, history=None, history_lens=None,
               prompt_lens=None, repetition=None, presence=None, frequency=None, bias_starts=None, bias_tokens=None,
               bias_values=None, allowed=None, allowed_rows=None, token_ids=None, ancestors=None, tokens=None,
               stream=None, prompt_nodes=None):
        """logits, out [T][vocab] (out may be logits): rows token_starts[b] .. token_starts[b+1] are request
        b's.  history [requests][longest] with history_lens: the requests' tokens, the first prompt_lens of
        them their prompts.  repetition, presence, frequency: float32, one a request.  bias_*: the entries of
        request b are bias_starts[b] .. bias_starts[b+1].  allowed: rows of 32 tokens a word, allowed_rows which
        of them is a row's (-1: none).  token_ids [T], ancestors [T][words]: a drafted tree's tokens, each row's
        way being part of its output (so that a history ends before the root); prompt_nodes [requests]: so many
        of the first nodes are the prompt's instead.  tokens (optional): int32 [T], the best token of each row
        or -1."""
        def refuse(why):
            raise TFError(TF_ERR_INVALID_ARG, "LogitRules.encode: " + why)

        i32, f32, place = torch.int32, torch.float32, self._place
        if logits.dim() != 2 or out.shape != logits.shape or out.dtype is not logits.dtype or logits.dtype not in _LOGITS:
            refuse("logits and out are [rows][vocab] of one float type")
        T, V = logits.shape
        if V > 1 and (logits.stride(1) != 1 or out.stride(1) != 1):
            refuse("rows must be contiguous")
        B = token_starts.numel() - 1
        d = LogitRulesDesc()
        if history is not None:
            if history_lens is None:
                refuse("a history has lengths")
            d.history, d.history_stride, d.max_history = self._matrix(history, B, "history"), history.stride(0), history.shape[1]
            d.history_lens = place(history_lens, i32, B, "history_lens")
            d.prompt_lens = place(prompt_lens, i32, B, "prompt_lens")
        elif history_lens is not None or prompt_lens is not None:
            refuse("lengths of no history")
        d.repetition = place(repetition, f32, B, "repetition")
        d.presence = place(presence, f32, B, "presence")
        d.frequency = place(frequency, f32, B, "frequency")
        if bias_starts is not None or bias_tokens is not None or bias_values is not None:
            if bias_starts is None or bias_tokens is None or bias_values is None:
                refuse("biases have starts, tokens and values")
            n = d.bias_count = bias_tokens.numel()
            d.bias_starts = place(bias_starts, i32, B + 1, "bias_starts")
            d.bias_tokens = place(bias_tokens, i32, n, "bias_tokens")
            d.bias_values = place(bias_values, f32, n, "bias_values")
        if allowed is not None:
            d.allowed, d.allowed_stride, d.allowed_count = self._matrix(allowed, -1, "allowed", -(-V // 32)), allowed.stride(0), allowed.shape[0]
            if allowed.shape[1] * 32 < V:
                refuse("allowed must have a bit for every token")
            d.allowed_rows = place(allowed_rows, i32, T, "allowed_rows")
            if not allowed.shape[0]:  # (an empty tensor is nowhere: a place that is not read, since no row is there)
                if T and allowed_rows is None:
                    refuse("a row of allowed tokens for every row")
                d.allowed, d.allowed_stride = d.allowed_rows, 0
        elif allowed_rows is not None:
            refuse("rows of no allowed tokens")
        if token_ids is not None or ancestors is not None:
            if token_ids is None or ancestors is None or ancestors.dim() != 2:
                refuse("drafted tokens and their ancestors [rows][words] go together")
            d.words = ancestors.shape[1]
            d.token_ids = place(token_ids, i32, T, "token_ids")
            d.ancestors = place(ancestors, i32, T * d.words, "ancestors")
            d.prompt_nodes = place(prompt_nodes, i32, B, "prompt_nodes")
        elif prompt_nodes is not None:
            refuse("a prompt among no drafted tokens")
        st = self.call(self.ctx.handle, self._here(logits, "logits"), logits.stride(0), self._here(out, "out"), out.stride(0),
                       _LOGITS[logits.dtype], V, T, place(token_starts, i32, B + 1, "token_starts"), B, max_query, C.byref(d),
                       place(tokens, i32, T, "tokens"), self._here(workspace, "workspace"), workspace.nbytes,
                       raw_stream(stream, self.ctx.device))
        if st:
            self.ctx.check(st, "LogitRules.encode")
