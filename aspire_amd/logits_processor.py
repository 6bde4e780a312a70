"""Logits processing on the HIP path: drop-in for the ``flashinfer.logits_processor`` pieces
the reference composes (aspire/models/sparse_draft_runner.py:527-554).

``LogitsPipe([Temperature(), Softmax(), TopP()])(values, temperature=..., top_p=...)`` runs
one kernel (``aspire_logits_pipe``): fp32 ``softmax(values / temperature)`` and top-p
renormalisation per row. ``define_logit_process_op`` registers ``mylib::logit_process``
around a pipe, as ``_define_logit_op`` does, with the fake (meta) implementation
torch.compile traces through.

``adjust_logits`` (not in the reference, whose pipes take logits as they are) goes before a pipe, a greedy pick or
``local_topk_candidates``: penalties for repeated tokens, biases (``LogitBias``) and grammar masks, one launch
(``aspire_adjust_logits``).
"""

from __future__ import annotations

import math
import struct

import torch
from torch.autograd import forward_ad

from aspire_amd import _lib


class Temperature:
    """Divide the values by ``temperature`` (a keyword of the pipe call)."""


class Softmax:
    """Softmax over the last dimension, in fp32."""


class TopP:
    """Top-p renormalisation with ``top_p`` (a keyword of the pipe call)."""


_ORDER = (Temperature, Softmax, TopP)


class LogitsPipe:
    """A sequence of the ops above; Softmax is required, Temperature may precede it and TopP
    follow it (the compositions the reference builds)."""

    def __init__(self, ops):
        kinds = [type(op) for op in ops]
        if Softmax not in kinds:
            raise ValueError("LogitsPipe needs a Softmax")
        idx = [_ORDER.index(k) if k in _ORDER else -1 for k in kinds]
        if -1 in idx or idx != sorted(idx) or len(set(idx)) != len(idx):
            raise ValueError("supported pipes: [Temperature()], Softmax(), [TopP()] in that order")
        self.ops = list(ops)
        self._temperature = Temperature in kinds
        self._top_p = TopP in kinds

    def __call__(self, values: torch.Tensor, temperature: float | None = None, top_p: float | None = None):
        if self._temperature and temperature is None:
            raise ValueError("this pipe applies Temperature: pass temperature=")
        if self._top_p and top_p is None:
            raise ValueError("this pipe applies TopP: pass top_p=")
        _lib.require_cuda(values, what="LogitsPipe")
        if values.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("values must be bf16 or fp32")
        shape = values.shape
        v = values if values.dim() == 2 else values.reshape(-1, shape[-1])
        if v.stride(-1) != 1:
            v = v.contiguous()
        rows, width = v.shape
        probs = torch.empty(shape, dtype=torch.float32, device=values.device)
        rc = _lib.lib().aspire_logits_pipe(
            _lib.ptr(v), 1 if v.dtype == torch.float32 else 0, v.stride(0), rows, width,
            float(temperature) if self._temperature else 0.0, float(top_p) if self._top_p else 0.0,
            _lib.ptr(probs), width, _lib.stream_of(values))
        _lib.check(rc, "LogitsPipe")
        return probs


def define_logit_process_op(pipe: LogitsPipe, kwargs: dict):
    """Register ``mylib::logit_process(Tensor vals) -> Tensor`` running ``pipe(vals, **kwargs)``
    (sparse_draft_runner.py:527-537); the fake implementation returns an fp32 tensor like vals."""
    torch.library.define("mylib::logit_process", "(Tensor vals) -> Tensor")

    @torch.library.impl("mylib::logit_process", "cuda")
    def _logit_process(vals):
        return pipe(vals, **kwargs)

    @torch.library.register_fake("mylib::logit_process")
    def _logit_process_fake(vals):
        return torch.empty_like(vals, dtype=torch.float32)

    return torch.ops.mylib.logit_process


def build_logits_pipe(temperature: float = 0, top_p: float = 0):
    """The pipe and keywords ``set_logit_processing`` builds: Temperature when temperature > 0,
    Softmax, TopP when top_p > 0."""
    ops, kwargs = [], {}
    if temperature > 0:
        ops.append(Temperature())
        kwargs["temperature"] = temperature
    ops.append(Softmax())
    if top_p > 0:
        ops.append(TopP())
        kwargs["top_p"] = top_p
    return LogitsPipe(ops), kwargs


class LogitBias:
    """Each request's biases (``{token: value}``, or None) on a device, for ``adjust_logits``; made when requests come or go."""

    def __init__(self, biases, device="cuda"):
        ids, values, ends = [], [], [0]
        for m in biases:
            start = len(ids)
            for token, given, value in sorted(((int(t), t, float(v)) for t, v in (m or {}).items())):
                if token != given or not 0 <= token < 1 << 31 or math.isnan(value):
                    raise ValueError("LogitBias: tokens must be whole numbers from 0 to 2^31 - 1, values not NaN")
                if len(ids) > start and ids[-1] == token:  # (keys that are not equal, tensors say, may name one token)
                    raise ValueError(f"LogitBias: two values for token {token}")
                ids.append(token)
                values.append(value)
            ends.append(len(ids))
        self.requests = len(ends) - 1
        self.ids = torch.tensor(ids, dtype=torch.int32, device=device)
        self.values = torch.tensor(values, dtype=torch.float32, device=device)
        self.indptr = torch.tensor(ends, dtype=torch.int32, device=device)


_LOGIT_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ADJUST = struct.Struct("PqPqPPqPPPPPPPqPPPPqPq8i")  # aspire_adjust_logits_args


def adjust_logits(logits: torch.Tensor, *, qo_indptr: torch.Tensor | None = None, history: torch.Tensor | None = None,
                  history_lens: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                  repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                  frequency: torch.Tensor | None = None, tree_tokens: torch.Tensor | None = None,
                  tree_masks: torch.Tensor | None = None, bias: LogitBias | None = None,
                  grammar: torch.Tensor | None = None, grammar_rows: torch.Tensor | None = None, vocab_start: int = 0,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Logits ``[T, V]`` (bf16, fp16 or fp32) with penalties for repeated tokens, biases and masks, as a new tensor or in
    ``out`` (which may be ``logits`` itself).

    Request ``b`` (of at most 65,535) has the rows ``qo_indptr[b]`` to ``qo_indptr[b + 1]`` (None: row ``b``, as many requests as
    rows); rows of no request are left as they were in ``out``. In this order, in fp32, rounded once:

    * ``x / repetition`` for ``x > 0``, else ``x * repetition``, for every token of the request's prompt or output; then
      ``x - frequency * count - presence * (count > 0)``, ``count`` its occurrences in the output (fp32 ``[B]`` each, None: 1, 0
      and 0). ``history`` int32 ``[B, H]`` holds ``history_lens[b]`` tokens, the first ``prompt_lens[b]`` the prompt's (None: none).
      With ``tree_tokens`` int32 ``[T]`` and ``tree_masks`` int64 ``[T, W]`` (as ``tree_attention`` takes them) the drafted tokens
      that a row sees, itself among them, are output too: they are then not in the history. Tokens outside the vocabulary do not count;
    * ``x + bias`` for the request's ``LogitBias`` entries;
    * ``-inf`` where the row's mask does not allow a token: bit ``i % 32`` of word ``i // 32`` of ``grammar`` int32 ``[G, ceil(V / 32)]``,
      row ``grammar_rows[t]`` (int32 ``[T]``; an index outside: no mask) or ``t``.

    ``vocab_start`` is the token of column 0, for a shard of the vocabulary; masks are the shard's. Not differentiable."""
    what = "adjust_logits"
    index, shape, st, dtype = logits.get_device(), logits.shape, logits.stride(), logits.dtype
    if index < 0:
        _lib.require_cuda(logits, what=what)
    floats = (logits, out, repetition, presence, frequency, None if bias is None else bias.values)
    if torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in floats]) \
            or forward_ad._current_level >= 0 and _lib.has_tangent(*floats):
        raise ValueError(f"{what}: not differentiable")
    code = _LOGIT_DTYPES.get(dtype)
    if code is None or len(shape) != 2 or (shape[1] > 1 and st[1] != 1):
        raise ValueError(f"{what}: logits must be bf16, fp16 or fp32 [T, V] with contiguous rows")
    tokens, vocab = shape
    device = logits.device
    if out is None:
        out, os = torch.empty((tokens, vocab), dtype=dtype, device=device), (vocab, 1)
    elif out is logits:
        os = st
    else:
        os = out.stride()
        if out.shape != shape or out.dtype is not dtype or out.get_device() != index or (vocab > 1 and os[1] != 1):
            raise ValueError(f"{what}: out must be of logits' shape and type on {device} with contiguous rows")
        if _lib.overlap(out, logits) and (out.data_ptr() != logits.data_ptr() or os != st):
            raise ValueError(f"{what}: out must be logits itself or apart from it")
    if tokens > 1 and os[0] < vocab:
        raise ValueError(f"{what}: the rows of out share memory")

    def vector(t, name, dtype, length=None, least=None):
        if t is None:
            return None
        if t.dtype is dtype and t.get_device() == index and t.dim() == 1 and t.is_contiguous() \
                and (length is None or t.shape[0] == length) and (least is None or t.shape[0] >= least):
            return t
        good = t.dim() == 1 and t.get_device() == index and (t.dtype == dtype or dtype is torch.int32 and t.dtype == torch.int64)
        if not good or length is not None and t.shape[0] != length or least is not None and t.shape[0] < least:
            raise ValueError(f"{what}: {name} must be {dtype} [{length if length is not None else f'at least {least or 0}'}] on {device}")
        return _lib.indices(t) if dtype is torch.int32 else _lib.dense(t, dtype)

    i32, f32 = torch.int32, torch.float32
    qo = vector(qo_indptr, "qo_indptr", i32, least=1)
    requests = tokens if qo is None else qo.shape[0] - 1
    lens = vector(history_lens, "history_lens", i32, requests)
    told = vector(prompt_lens, "prompt_lens", i32, requests)
    rep = vector(repetition, "repetition", f32, requests)
    pres = vector(presence, "presence", f32, requests)
    freq = vector(frequency, "frequency", f32, requests)
    history_stride = history_len = mask_stride = words = grammar_stride = grammar_count = 0
    if history is not None:
        if history.dim() != 2 or history.dtype is not i32 or history.shape[0] != requests or history.get_device() != index \
                or (history.shape[1] > 1 and history.stride(1) != 1) or lens is None:
            raise ValueError(f"{what}: history must be int32 [{requests}, H] on {device} with contiguous rows, and history_lens given")
        history_stride, history_len = history.stride(0), history.shape[1]
    elif lens is not None or told is not None:
        raise ValueError(f"{what}: history_lens and prompt_lens go with history")
    if (tree_tokens is None) != (tree_masks is None) or tree_masks is not None and qo is None:
        raise ValueError(f"{what}: tree_tokens and tree_masks go together, with qo_indptr")
    tree = vector(tree_tokens, "tree_tokens", i32, least=tokens)
    if tree_masks is not None:
        if tree_masks.dtype != torch.int64 or tree_masks.dim() != 2 or tree_masks.shape[0] < tokens or tree_masks.get_device() != index \
                or (tree_masks.shape[1] > 1 and tree_masks.stride(1) != 1):
            raise ValueError(f"{what}: tree_masks must be int64 [T, words] on {device} with contiguous rows")
        mask_stride, words = tree_masks.stride(0), tree_masks.shape[1]
    if (history is not None or tree is not None) and rep is None and pres is None and freq is None:
        raise ValueError(f"{what}: a history or a tree needs repetition, presence or frequency")
    if history is None and tree is None and (rep is not None or pres is not None or freq is not None):
        raise ValueError(f"{what}: penalties need a history or a tree")
    if bias is not None and (bias.requests != requests or bias.indptr.get_device() != index):
        raise ValueError(f"{what}: bias must hold {requests} requests on {device}")
    if grammar is not None:
        if grammar.dtype != i32 or grammar.dim() != 2 or grammar.shape[1] < (vocab + 31) // 32 or grammar.get_device() != index \
                or (grammar.shape[1] > 1 and grammar.stride(1) != 1) or (grammar_rows is None and grammar.shape[0] < tokens):
            raise ValueError(f"{what}: grammar must be int32 [rows, {(vocab + 31) // 32}] on {device} with contiguous rows, a row for each "
                             "row of logits or grammar_rows given")
        grammar_stride, grammar_count = grammar.stride(0), grammar.shape[0]
    elif grammar_rows is not None:
        raise ValueError(f"{what}: grammar_rows go with grammar")
    which = vector(grammar_rows, "grammar_rows", i32, least=tokens)
    if not 0 <= vocab_start <= (1 << 31) - vocab:
        raise ValueError(f"{what}: the shard's tokens must lie in 0 to 2^31 - 1")
    if not words:  # no drafted token is on a path (and masks without words have no address)
        tree = tree_masks = None
    at = lambda t: 0 if t is None else t.data_ptr()
    b = (None, None, None) if bias is None else (bias.ids, bias.values, bias.indptr)
    args = _ADJUST.pack(logits.data_ptr(), st[0], out.data_ptr(), os[0], at(qo), at(history), history_stride,
                        at(lens), at(told), at(rep), at(pres), at(freq), at(tree), at(tree_masks), mask_stride, at(b[0]), at(b[1]),
                        at(b[2]), at(grammar), grammar_stride, at(which), vocab_start, tokens, vocab, requests, code, history_len,
                        words, grammar_count, 0 if bias is None else bias.ids.shape[0])
    _lib.launch(_lib.lib().aspire_adjust_logits, index, what, args)
    return out


__all__ = ["LogitBias", "adjust_logits", "LogitsPipe", "Temperature", "Softmax", "TopP", "define_logit_process_op", "build_logits_pipe"]
