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
from .kv_cache import _FLOAT_CODES, _has_tangent

_MAX_CHECKED = 64


class _WithoutGradient(torch.autograd.Function):
    """Scores as they are; a backward pass that reaches them, or a tangent, is told that it ends there."""

    @staticmethod
    def forward(ctx, out, *inputs):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, *gradients):
        raise RuntimeError("beam_select has no gradient: detach its logits and scores, or call it under torch.no_grad()")

    @staticmethod
    def jvp(ctx, *tangents):
        raise RuntimeError("beam_select has no gradient, nor a tangent: detach its logits and scores")


class BeamOps:
    """The entry point, part of ``HipRNSBackend``."""

    def beam_select(self, logits: torch.Tensor, scores: torch.Tensor, k: int, *, finished: torch.Tensor | None = None,
                    end_token: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The ``k`` best continuations of each request's beams, best first, in one launch for
        up to 16384 requests.

        ``logits`` ``[requests, beams, vocabulary]`` (rows of any strides), ``scores``
        float32 ``[requests, beams]``, each beam's so far.  A continuation's score is its beam's
        plus the token's log-probability (``log_softmax`` over the vocabulary); of equal ones
        the lower beam's goes first, within a beam the larger logit, then the lower token.
        Exponentials are float32, log-sums and scores 64 bits: a log-sum is off by up to
        ``(3 ln(vocabulary + 1) + 35) 2**-24``.  The order is exact within a beam and among beams
        of the same logits; other beams' continuations nearer than twice that may come in
        either order (and in another where a call has more requests).  A beam that is ``finished`` (bool ``[requests, beams]``) goes on
        as it is, once, with ``end_token``; its logits are not read.  A logit or score of
        minus infinity is no candidate; a beam whose logits hold a NaN or plus infinity has none.

        -> float32 scores, int32 tokens and int32 parents ``[requests, k]``, a parent being
        ``request * beams + beam``.  A place that no candidate is left for has score minus
        infinity, ``end_token`` (0 without one) and its own number modulo the beams as its
        parent's.  ``k`` and ``beams`` are at most 64, ``beams * ceil(vocabulary / 16384)`` 1024.
        There is no gradient: a backward pass through the scores raises, a call with a tangent too."""
        k = operator.index(k)
        end_token = None if end_token is None else operator.index(end_token)
        key = (logits.dtype, logits.shape, logits.stride(), logits.device, scores.dtype, scores.shape, scores.stride(), scores.device,
               k, None if finished is None else (finished.dtype, finished.shape, finished.stride(), finished.device), end_token)
        checked = self._beam_checked.get(key)
        if checked is None:
            plain = self._plain_beams(logits, scores, k, finished, end_token)
            if any(x is not y for x, y in zip(plain, (logits, scores, finished))):
                return self.beam_select(plain[0], plain[1], k, finished=plain[2], end_token=end_token)
            checked = self._beam_call(logits, k, end_token)
            if len(self._beam_checked) >= _MAX_CHECKED:
                self._beam_checked.clear()
            self._beam_checked[key] = checked
        _, ref, need, like = checked
        device = logits.device
        space = self._kv_scratch_for(need, device, self._stream_of(device))
        out = torch.empty_like(like[0], memory_format=torch.contiguous_format)
        tokens = torch.empty_like(like[1], memory_format=torch.contiguous_format)
        parents = torch.empty_like(like[1], memory_format=torch.contiguous_format)
        self._on_device(device, self._lib.rnsmx_beam_select, ref, logits.data_ptr(), scores.data_ptr(),
                        None if finished is None else finished.data_ptr(), space.data_ptr(), space.numel(), out.data_ptr(),
                        tokens.data_ptr(), parents.data_ptr())
        self._stats["beam_select_calls"] += 1
        if torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad) or _has_tangent(logits, scores):
            out = _WithoutGradient.apply(out, logits, scores)
        return out, tokens, parents

    @staticmethod
    def _plain_beams(logits: torch.Tensor, scores: torch.Tensor, k: int, finished: torch.Tensor | None, end_token: int | None):
        """The checked tensors as the library takes them: values of a row, scores and flags side by side."""
        if logits.dtype not in _FLOAT_CODES or logits.ndim != 3:
            raise ValueError("logits must be [requests, beams, vocabulary] in float32, float16 or bfloat16")
        requests, beams, vocabulary = logits.shape
        device = logits.device
        if scores.dtype != torch.float32 or scores.shape != (requests, beams) or scores.device != device:
            raise ValueError(f"scores must be float32 [{requests}, {beams}] on {device}")
        if not 1 <= beams <= _native.BEAMS_MAX or not 1 <= k <= _native.BEAMS_MAX:
            raise ValueError(f"1 to {_native.BEAMS_MAX} beams and continuations, got {beams} and {k}")
        if vocabulary < 1:
            raise ValueError("a vocabulary has at least one token")
        if finished is not None:
            if finished.dtype != torch.bool or finished.shape != scores.shape or finished.device != device:
                raise ValueError(f"finished must be bool [{requests}, {beams}] on {device}")
            if end_token is None:
                raise ValueError("finished beams need an end_token")
        if end_token is not None and not 0 <= end_token < vocabulary:
            raise ValueError(f"end_token must be a token of the vocabulary, got {end_token}")
        if device.type != "cuda":
            raise ValueError(f"logits must be on the GPU, they are on {device}")
        return (logits if logits.stride(2) == 1 else logits.contiguous(), scores if scores.is_contiguous() else scores.contiguous(),
                finished if finished is None or finished.is_contiguous() else finished.contiguous())

    def _beam_call(self, logits: torch.Tensor, k: int, end_token: int | None):
        requests, beams, vocabulary = logits.shape
        struct = _native.BeamsStruct(logits.stride(0), logits.stride(1), _FLOAT_CODES[logits.dtype], requests, beams, vocabulary, k,
                                     -1 if end_token is None else end_token)
        ref = ctypes.addressof(struct)
        need = int(self._lib.rnsmx_beam_workspace_bytes(ref))
        if need < 0:
            _native.check(_native.EINVAL)
        # one number's memory in the outputs' shape: what they are made like costs less than their sizes
        like = tuple(torch.empty((1,), dtype=dtype, device=logits.device).expand(requests, k)
                     for dtype in (torch.float32, torch.int32))
        return struct, ref, need, like
