"""A model's logits made ready for the choice of a token, on the GPU.

``adjust_logits`` applies what a request asks of its next token in one pass over the logits
(``wn_adjust_logits``): penalties for tokens that its history holds, biases of single tokens,
and a bit mask of the tokens that a grammar allows. The engine's requests reach it through
their ``repetition_penalty``, ``presence_penalty``, ``frequency_penalty``, ``logit_bias`` and
``allowed_tokens``. There is no host fallback."""
from __future__ import annotations

import ctypes
import math

import torch

from winnow_amd import _lib
from winnow_amd.packed_attention import UnsupportedLayout, values_only

MAX_BIASES = 1024          # entries of a row's bias list
MAX_HISTORY = 2 ** 30 - 1  # tokens of a row's history


def mask_words(vocab: int) -> int:
    """32-bit words of a row of ``allowed`` over ``vocab`` tokens."""
    return -(-vocab // 32)


def pack_allowed(allowed: torch.Tensor) -> torch.Tensor:
    """(..., V) truth values -> (..., mask_words(V)) int32, bit v % 32 of word v // 32."""
    V = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed.to(torch.int64), (0, 32 * mask_words(V) - V)).unflatten(-1, (-1, 32))
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def fp32(value) -> float:
    """What a number becomes in the type that it is applied in: infinite past fp32's range, 0 below it."""
    try:
        return ctypes.c_float(float(value)).value
    except OverflowError:
        return math.inf if value > 0 else -math.inf


def _penalty(name: str, value, N: int, device: torch.device) -> tuple:
    """(tensor or None, scalar) of a penalty given as a number or one per row."""
    if not isinstance(value, torch.Tensor):
        if type(value) is float and (value == 0.0 if name != "repetition" else value == 1.0):
            return None, value
        value = fp32(value)
        if not math.isfinite(value) or (name == "repetition" and value <= 0):
            raise UnsupportedLayout(f"{name} must be finite{' and above 0' if name == 'repetition' else ''} in fp32, got {value} there")
        return None, value
    if value.shape != (N,) or value.dtype != torch.float32 or value.device != device or not value.is_contiguous():
        raise UnsupportedLayout(f"{name} must be a number or ({N},) fp32 on {device}, contiguous, got "
                                f"{tuple(value.shape)} {value.dtype} on {value.device}")
    return value, 0.0


def _whole(name: str, t: torch.Tensor, shape: tuple, device: torch.device) -> torch.Tensor:
    """An integer operand as int32 with a contiguous last axis."""
    if t.shape != shape or t.dtype not in (torch.int32, torch.int64) or t.device != device:
        raise UnsupportedLayout(f"{name} must be {shape} int32 (or int64) on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if t.dtype == torch.int64:
        # of no vocabulary and no length that is served, and so where the type holds them
        t = t.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def adjust_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                  prompt_lengths: torch.Tensor | None = None, repetition=1.0, presence=0.0, frequency=0.0,
                  bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  allowed: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``logits`` (N, V), fp32/fp16/bf16 with a contiguous last axis and any row stride -> the
    adjusted logits, (N, V) of the same type: a new tensor, or ``out`` (which may be ``logits``).

    For each row, in this order:

    * ``history`` (N, H) int32 are its tokens so far, of which the first ``lengths`` (N,) count
      (all H without it). A token that occurs has its logit divided by ``repetition`` where it is
      positive and multiplied by it elsewhere. Of those from ``prompt_lengths`` (N,) on (0 without
      it: all), one that occurs c > 0 times loses ``frequency`` c + ``presence``. The penalties are
      numbers (finite in fp32, ``repetition`` above 0) or (N,) fp32. Tokens outside [0, V) are ignored.
    * ``bias`` (N, J) fp32 is added to the logits of the tokens ``bias_ids`` (N, J), J <= 1024; ids
      outside [0, V) pad the list; a token listed more than once gets each of its biases, in order.
    * ``allowed`` (N, ceil(V / 32)) int32: the logit of token v becomes -inf where bit v % 32 of
      word v // 32 is 0 (``pack_allowed``). A row that allows nothing is -inf everywhere.

    The arithmetic is fp32, rounded once to the logits' type; a logit that nothing applies to
    keeps its bits. Integer operands may be int64 (copied). Raises ``UnsupportedLayout`` before
    the launch for tensors off the GPU, of other types or shapes, or where a gradient, a tangent
    or a trace is asked for."""
    if not _lib.is_hip(logits):
        raise UnsupportedLayout("adjust_logits needs logits on a HIP device; there is no host fallback")
    if logits.dtype not in _lib.DTYPE_CODE or logits.dim() != 2:
        raise UnsupportedLayout(f"logits must be (N, V) of fp32, fp16 or bf16, got {tuple(logits.shape)} {logits.dtype}")
    (N, V), dev = logits.shape, logits.device
    if not 1 <= V <= 2 ** 31 - 1 - 65536 or (V > 1 and logits.stride(1) != 1):
        raise UnsupportedLayout(f"logits need a contiguous, non-empty last axis of fewer than 2^31 - 65536, got {V}")
    values_only("adjust_logits", *[t for t in (logits, bias, repetition, presence, frequency, out) if isinstance(t, torch.Tensor)])
    if history is None and (lengths is not None or prompt_lengths is not None):
        raise UnsupportedLayout("lengths and prompt_lengths are those of a history")
    H = 0
    if history is not None:
        if history.dim() != 2 or history.shape[1] > MAX_HISTORY:
            raise UnsupportedLayout(f"history must be ({N}, H), H <= {MAX_HISTORY}, got {tuple(history.shape)}")
        H = history.shape[1]
        history = _whole("history", history, (N, H), dev)
        if lengths is not None:
            lengths = _whole("lengths", lengths, (N,), dev)
        if prompt_lengths is not None:
            prompt_lengths = _whole("prompt_lengths", prompt_lengths, (N,), dev)
    rep = _penalty("repetition", repetition, N, dev)
    pres, freq = _penalty("presence", presence, N, dev), _penalty("frequency", frequency, N, dev)
    if (bias is None) != (bias_ids is None):
        raise UnsupportedLayout("bias and bias_ids come together")
    J = 0
    if bias is not None:
        if bias.dim() != 2 or bias.shape[0] != N or bias.shape[1] > MAX_BIASES or bias.dtype != torch.float32 or bias.device != dev:
            raise UnsupportedLayout(f"bias must be ({N}, J) fp32 on {dev}, J <= {MAX_BIASES}, got {tuple(bias.shape)} {bias.dtype} on {bias.device}")
        J = bias.shape[1]
        bias_ids = _whole("bias_ids", bias_ids, (N, J), dev)
        bias = bias if J <= 1 or bias.stride(1) == 1 else bias.contiguous()
    words = (V + 31) // 32
    if allowed is not None and (allowed.shape != (N, words) or allowed.dtype != torch.int32 or allowed.device != dev
                                or (words > 1 and allowed.stride(1) != 1)):
        raise UnsupportedLayout(f"allowed must be ({N}, {words}) int32 on {dev} with contiguous rows, got "
                                f"{tuple(allowed.shape)} {allowed.dtype} on {allowed.device}")
    if out is None:
        out = torch.empty(N, V, dtype=logits.dtype, device=dev)
    elif out.shape != (N, V) or out.dtype != logits.dtype or out.device != dev or (V > 1 and out.stride(1) != 1) \
            or (N > 1 and out.stride(0) < V):
        raise UnsupportedLayout(f"out must be ({N}, {V}) {logits.dtype} on {dev} with contiguous rows of its own")
    elif _shares(out, logits) and (out.data_ptr() != logits.data_ptr() or (N > 1 and out.stride(0) != logits.stride(0))):
        raise UnsupportedLayout("out may be logits itself, but no other view of its memory")
    elif any(t is not None and _shares(out, t) for t in (history, lengths, prompt_lengths, rep[0], pres[0], freq[0], bias_ids, bias, allowed)):
        raise UnsupportedLayout("out shares memory with another operand")
    if N == 0:
        return out
    (rep_t, rep_x), (pres_t, pres_x), (freq_t, freq_x) = rep, pres, freq
    with _lib.on(dev):
        _lib.call("wn_adjust_logits", logits.data_ptr(), _lib.DTYPE_CODE[logits.dtype], logits.stride(0), out.data_ptr(), out.stride(0), N, V,
                  None if history is None else history.data_ptr(), history.stride(0) if H else 0, H,
                  None if lengths is None else lengths.data_ptr(), None if prompt_lengths is None else prompt_lengths.data_ptr(),
                  None if rep_t is None else rep_t.data_ptr(), None if pres_t is None else pres_t.data_ptr(),
                  None if freq_t is None else freq_t.data_ptr(), rep_x, pres_x, freq_x,
                  None if bias is None else bias_ids.data_ptr(), bias_ids.stride(0) if J else 0,
                  None if bias is None else bias.data_ptr(), bias.stride(0) if J else 0, J,
                  None if allowed is None else allowed.data_ptr(), 0 if allowed is None else allowed.stride(0), _lib.stream_of(dev))
    return out


def _shares(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory that the two tensors span overlaps."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1
