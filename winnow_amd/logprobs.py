"""Log probabilities of tokens under a model's logits, on the GPU.

``token_logprobs`` reads every row of logits once (``wn_token_logprobs``) and gives, per
row, the log probability of a given token, the entropy of the distribution and the most
likely alternatives. It scores what an engine generates (``Request.top_logprobs``) and the
drafted tokens of a speculative step. There is no host fallback."""
from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from winnow_amd import _lib
from winnow_amd.packed_attention import UnsupportedLayout, values_only

MAX_TOP = 64


@dataclass
class TokenLogprobs:
    """Results of ``token_logprobs``; the shapes are the rows' (``logits.shape[:-1]``)."""

    logprob: torch.Tensor | None        # fp32; None without tokens
    entropy: torch.Tensor               # fp32, in nats
    top_logprobs: torch.Tensor | None   # (..., top) fp32, the most likely first; None for top = 0
    top_ids: torch.Tensor | None        # (..., top) int64; equal logits by the lowest index


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(rows: int, vocab: int, top: int) -> int:
    return int(_lib.lib().wn_token_logprobs_workspace_bytes(rows, vocab, top))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, top: int = 0) -> TokenLogprobs:
    """``logits`` (V,), (N, V) or (B, T, V), fp32/fp16/bf16 with a contiguous last axis and any
    other strides; ``tokens`` int64 (or int32) of the rows' shape; ``top`` 0 .. 64 alternatives.

    Sums are fp32 whatever the logits' type. A logit of -inf has probability 0; a row with a
    NaN or +inf, or without a finite logit, gives NaN (its ``top_ids`` still lie in [0, V));
    a token outside [0, V) gives NaN for its row. Raises ``UnsupportedLayout`` before the
    launch for tensors off the GPU, of other types or shapes, or where a gradient, a tangent or a
    trace is asked for."""
    if not _lib.is_hip(logits):
        raise UnsupportedLayout("token_logprobs needs logits on a HIP device; there is no host fallback")
    if logits.dtype not in _lib.DTYPE_CODE or not 1 <= logits.dim() <= 3:
        raise UnsupportedLayout(f"logits must be (V,), (N, V) or (B, T, V) of fp32, fp16 or bf16, got "
                                f"{tuple(logits.shape)} {logits.dtype}")
    values_only("token_logprobs", logits)
    rows, V = logits.shape[:-1], logits.shape[-1]
    if not 1 <= V < 2 ** 31 or (V > 1 and logits.stride(-1) != 1):
        raise UnsupportedLayout(f"logits need a contiguous, non-empty last axis of fewer than 2^31, got {V}")
    if not 0 <= top <= min(MAX_TOP, V):
        raise UnsupportedLayout(f"top {top} must be 0 .. {MAX_TOP} and at most the {V} logits of a row")
    if tokens is not None:
        if tokens.shape != rows or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != logits.device:
            raise UnsupportedLayout(f"tokens must be {tuple(rows)} int64 on {logits.device}, got "
                                    f"{tuple(tokens.shape)} {tokens.dtype} on {tokens.device}")
        if tokens.dtype != torch.int64 or not tokens.is_contiguous():
            tokens = tokens.to(torch.int64).contiguous()
    N = rows.numel()
    dev = logits.device
    new = torch.empty((2 if tokens is not None else 1, *rows), dtype=torch.float32, device=dev)
    entropy, logprob = new[0], new[1] if tokens is not None else None
    top_lp = torch.empty(*rows, top, dtype=torch.float32, device=dev) if top else None
    top_id = torch.empty(*rows, top, dtype=torch.int64, device=dev) if top else None
    result = TokenLogprobs(logprob, entropy, top_lp, top_id)
    if N == 0:
        return result
    st = logits.stride()
    outer, inner, n_inner = (st[0], st[1], rows[1]) if len(rows) == 2 else (0, st[0] if rows else 0, N)
    need = _workspace_bytes(N, V, top)
    workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _lib.on(dev):
        _lib.call("wn_token_logprobs", _lib.ptr(logits), _lib.DTYPE_CODE[logits.dtype], outer, inner, n_inner,
                  _lib.ptr(tokens), _lib.ptr(logprob), _lib.ptr(entropy), _lib.ptr(top_lp), _lib.ptr(top_id), N, V, top,
                  _lib.ptr(workspace), need, _lib.stream_of(dev))
    return result
