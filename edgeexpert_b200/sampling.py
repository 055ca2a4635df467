"""Output-head sampling, mirroring the reference's LogitSoftcapSoftmax,
Sample and SampleTopK64 encoders (Kernels/Sampling/LogitOutput.swift;
Metal/Sampling/logit.metal:42-617) on libtfcuda.so; and, without a counterpart
there, LogitRules: penalties, biases and grammar masks on the logits of a
ragged batch before any of them."""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import (Context, LogitRulesDesc, TF_ERR_INVALID_ARG, TFError, lib, on_device, ptr, stream_ptr)

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

    @staticmethod
    def _vectors(n: int, dtype, what: str, *tensors):
        for t in tensors:
            if t is not None and (t.dtype is not dtype or t.numel() != n or not t.is_contiguous()):
                raise TFError(TF_ERR_INVALID_ARG, f"LogitRules.encode: {what}: {n} contiguous values of {dtype}")

    @staticmethod
    def _matrix(t, rows, what: str):
        if t.dtype is not torch.int32 or t.dim() != 2 or (rows is not None and t.shape[0] != rows) or (
                t.shape[1] > 1 and t.stride(1) != 1):
            raise TFError(TF_ERR_INVALID_ARG, f"LogitRules.encode: {what} must be an int32 matrix, rows contiguous")

    def encode(self, logits, out, token_starts, workspace, max_query: int = 1, history=None, history_lens=None,
               prompt_lens=None, repetition=None, presence=None, frequency=None, bias_starts=None, bias_tokens=None,
               bias_values=None, allowed=None, allowed_rows=None, token_ids=None, ancestors=None, tokens=None,
               stream=None):
        """logits, out [T][vocab] (out may be logits): rows token_starts[b] .. token_starts[b+1] are request
        b's.  history [requests][longest] with history_lens: the requests' tokens, the first prompt_lens of
        them their prompts.  repetition, presence, frequency: float32, one a request.  bias_*: the entries of
        request b are bias_starts[b] .. bias_starts[b+1].  allowed: rows of 32 tokens a word, allowed_rows which
        of them is a row's (-1: none).  token_ids [T], ancestors [T][words]: a drafted tree's tokens, each row's
        way being part of its output.  tokens (optional): int32 [T], the best token of each row or -1."""
        what, i32 = "LogitRules.encode", torch.int32
        if logits.dim() != 2 or out.shape != logits.shape or out.dtype is not logits.dtype or logits.dtype not in _LOGITS:
            raise TFError(TF_ERR_INVALID_ARG, f"{what}: logits and out are [rows][vocab] of one float type")
        T, V = logits.shape
        if V > 1 and (logits.stride(1) != 1 or out.stride(1) != 1):
            raise TFError(TF_ERR_INVALID_ARG, f"{what}: rows must be contiguous")
        B = token_starts.numel() - 1
        self._vectors(B + 1, i32, "token_starts and bias_starts", token_starts, bias_starts)
        self._vectors(B, i32, "history_lens and prompt_lens", history_lens, prompt_lens)
        self._vectors(B, torch.float32, "repetition, presence and frequency", repetition, presence, frequency)
        self._vectors(T, i32, "allowed_rows, token_ids and tokens", allowed_rows, token_ids, tokens)
        on_device(what, self.ctx.device, logits, out, token_starts, workspace, history, history_lens, prompt_lens,
                  repetition, presence, frequency, bias_starts, bias_tokens, bias_values, allowed, allowed_rows,
                  token_ids, ancestors, tokens)
        if (history is None) != (history_lens is None) or (prompt_lens is not None and history is None):
            raise TFError(TF_ERR_INVALID_ARG, f"{what}: a history and its lengths go together")
        if (bias_starts is None) != (bias_tokens is None) or (bias_tokens is None) != (bias_values is None):
            raise TFError(TF_ERR_INVALID_ARG, f"{what}: biases have starts, tokens and values")
        if (token_ids is None) != (ancestors is None):
            raise TFError(TF_ERR_INVALID_ARG, f"{what}: drafted tokens and their ancestors go together")
        if allowed_rows is not None and allowed is None:
            raise TFError(TF_ERR_INVALID_ARG, f"{what}: rows of no allowed tokens")

        def at(t):
            return None if t is None else t.data_ptr()

        d = LogitRulesDesc(at(history), at(history_lens), at(prompt_lens), at(repetition), at(presence), at(frequency),
                           at(bias_starts), at(bias_tokens), at(bias_values), at(allowed), at(allowed_rows),
                           at(token_ids), at(ancestors))
        if history is not None:
            self._matrix(history, B, "history")
            d.history_stride, d.max_history = history.stride(0), history.shape[1]
        if bias_tokens is not None:
            n = bias_tokens.numel()
            self._vectors(n, i32, "bias_tokens", bias_tokens)
            self._vectors(n, torch.float32, "bias_values", bias_values)
            d.bias_count = n
        if allowed is not None:
            self._matrix(allowed, None, "allowed")
            if allowed.shape[1] * 32 < V:
                raise TFError(TF_ERR_INVALID_ARG, f"{what}: allowed must have a bit for every token")
            d.allowed_stride, d.allowed_count = allowed.stride(0), allowed.shape[0]
        if ancestors is not None:
            if ancestors.dtype is not i32 or ancestors.dim() != 2 or ancestors.shape[0] != T or not ancestors.is_contiguous():
                raise TFError(TF_ERR_INVALID_ARG, f"{what}: ancestors are a contiguous int32 [rows][words]")
            d.words = ancestors.shape[1]
        st = self.call(self.ctx.handle, logits.data_ptr(), logits.stride(0), out.data_ptr(), out.stride(0),
                       _LOGITS[logits.dtype], V, T, token_starts.data_ptr(), B, max_query, C.byref(d), at(tokens),
                       workspace.data_ptr(), workspace.nbytes, stream_ptr(stream))
        self.ctx.check(st, what)
