"""Beam search's selection over beams and vocabulary.

``beam_select`` takes the logits of every request's beams and gives the best
continuations, whose parents ``kv_reorder`` takes.  No counterpart in the
reference, which ends with the projections.
"""
from __future__ import annotations

import ctypes
import operator

import torch

from .. import _native
from .kv_cache import _FLOAT_CODES


class _WithoutGradient(torch.autograd.Function):
    """Scores as they are; a backward pass that reaches them says that it ends there."""

    @staticmethod
    def forward(ctx, out, *inputs):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, *gradients):
        raise RuntimeError("beam_select has no gradient: detach its logits and scores, or call it under torch.no_grad()")


class BeamOps:
    """The entry point, part of ``HipRNSBackend``."""

    def beam_select(self, logits: torch.Tensor, scores: torch.Tensor, k: int, *, finished: torch.Tensor | None = None,
                    end_token: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The ``k`` best continuations of each request's beams, best first, in one launch.

        ``logits`` ``[requests, beams, vocabulary]`` (rows of any strides), ``scores``
        float32 ``[requests, beams]``, each beam's so far.  A continuation's score is its beam's
        plus the token's log-probability (``log_softmax`` over the vocabulary), compared in
        64 bits; of equal ones the lower beam's goes first, within a beam the larger logit,
        then the lower token.  A beam that is ``finished`` (bool ``[requests, beams]``) goes on
        as it is, once, with ``end_token``; its logits are not read.  A logit or score of
        minus infinity is no candidate; a beam whose logits hold a NaN or plus infinity has none.

        -> float32 scores, int32 tokens and int32 parents ``[requests, k]``, a parent being
        ``request * beams + beam``.  A place that no candidate is left for has score minus
        infinity, ``end_token`` (0 without one) and its own number modulo the beams as its
        parent's.  There is no gradient: a backward pass through the scores raises."""
        k = operator.index(k)
        if logits.dtype not in _FLOAT_CODES or logits.ndim != 3:
            raise ValueError("logits must be [requests, beams, vocabulary] in float32, float16 or bfloat16")
        requests, beams, vocabulary = logits.shape
        device = logits.device
        if scores.dtype != torch.float32 or scores.shape != (requests, beams) or scores.device != device:
            raise ValueError(f"scores must be float32 [{requests}, {beams}] on {device}")
        if not 1 <= beams <= _native.BEAMS_MAX or not 1 <= k <= _native.BEAMS_MAX:
            raise ValueError(f"1 to {_native.BEAMS_MAX} beams and continuations, got {beams} and {k}")
        if finished is not None:
            if finished.dtype != torch.bool or finished.shape != scores.shape or finished.device != device:
                raise ValueError(f"finished must be bool [{requests}, {beams}] on {device}")
            if end_token is None:
                raise ValueError("finished beams need an end_token")
        if end_token is not None and not 0 <= end_token < vocabulary:
            raise ValueError(f"end_token must be a token of the vocabulary, got {end_token}")
        if device.type != "cuda":
            raise ValueError(f"logits must be on the GPU, they are on {device}")
        wanted = torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad)
        rows = logits if logits.stride(2) == 1 or vocabulary == 1 else logits.contiguous()
        plain = scores if scores.is_contiguous() else scores.contiguous()
        if finished is not None and not finished.is_contiguous():
            finished = finished.contiguous()
        struct = _native.BeamsStruct(rows.stride(0), rows.stride(1), _FLOAT_CODES[logits.dtype], requests, beams, vocabulary, k,
                                     -1 if end_token is None else int(end_token))
        ref = ctypes.addressof(struct)
        need = int(self._lib.rnsmx_beam_workspace_bytes(ref))
        if need < 0:
            _native.check(_native.EINVAL)
        space = self._kv_scratch_for(need, device, self._stream_of(device))
        out = torch.empty((requests, k), dtype=torch.float32, device=device)
        tokens = torch.empty((requests, k), dtype=torch.int32, device=device)
        parents = torch.empty_like(tokens)
        self._on_device(device, self._lib.rnsmx_beam_select, ref, rows.data_ptr(), plain.data_ptr(),
                        None if finished is None else finished.data_ptr(), space.data_ptr(), space.numel(), out.data_ptr(),
                        tokens.data_ptr(), parents.data_ptr())
        self._stats["beam_select_calls"] += 1
        return (_WithoutGradient.apply(out, logits, scores) if wanted else out), tokens, parents
