"""Decode-step token selection on the GPU: the reference's ``SamplingPolicy``
and ``TokenSampler`` (runtime/fast_decode.py:20-95) on one HIP kernel each.

Greedy selection runs ``koemi_herm_greedy_tokens`` (the padding id masked, the
first maximum winning, as ``argmax`` after ``index_fill`` does). Sampling runs
``koemi_herm_sample_tokens``: the padding id removed, the top-k restriction
(every score below the k-th largest set to -inf, ties kept), ``softmax(scores
/ temperature)``, then an inverse-CDF draw from a uniform number per row that
this front draws with ``torch.rand`` from the sampler's generator (the
reference draws with ``torch.multinomial``; the kernel takes the uniforms as
an input so that a captured decode graph can draw from numbers written into
a static buffer before each replay). Nothing is read back to the host.

``sample_tokens`` is the draw for any vocabulary, with top-p and min-p as well
(``koemi_sample_filtered``); a policy that names one of them, or logits wider than
``koemi_herm_sample_tokens`` takes, run it.
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch
from torch import Tensor

from koemi_amd import _native

__all__ = ["PAD_TOKEN_ID", "SamplingPolicy", "TokenSampler", "sample_tokens"]

PAD_TOKEN_ID = 256  # configuration/settings.py:10-11
_NARROW = 4096  # columns that koemi_herm_sample_tokens takes
_MAX_VOCAB = 1 << 19
_LOGIT_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


@lru_cache(maxsize=256)
def _workspace_bytes(rows: int, vocab: int) -> int:
    return _native.query("koemi_sample_filtered_workspace_bytes", rows, vocab)


def _check_share(name: str, value: float | None, zero: bool) -> None:
    if value is not None and (isinstance(value, bool) or not isinstance(value, (int, float))
                              or not (0.0 <= value <= 1.0 if zero else 0.0 < value <= 1.0)):
        raise ValueError(f"{name} must be a number {'from' if zero else 'above'} 0 and at most 1")


def sample_tokens(logits: Tensor, uniforms: Tensor, *, temperature: float = 1.0, top_k: int | None = None,
                  top_p: float | None = None, min_p: float | None = None, exclude: int | None = None,
                  with_probabilities: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """Ids drawn from ``[rows, vocabulary]`` logits with a uniform number in [0, 1) a row.

    ``logits`` float32, float16 or bfloat16 (rows with contiguous columns are read in place),
    at most 2^19 columns; ``uniforms`` ``[rows]`` float32. With w = exp((z - max z) /
    temperature): ``top_k`` keeps the k largest scores and the equals of the last;
    ``top_p`` of those the ids whose strictly better ones hold less than that share of their
    sum (so that equals stay together, and the share is reached); ``min_p`` of those the ones with w
    >= min_p. ``exclude`` (an id), -inf and NaN are never drawn; a row with +inf draws among
    those. The id is the first whose running sum of kept w, in the ids' order, exceeds uniform times
    the whole. Returns ``[rows, 1]`` int64 ids (0 for a row without a score) and, with
    ``with_probabilities``, the float32 distribution they come from. Weights are formed in
    64 bits and added as whole numbers, so results do not depend on an order. Nothing is
    read back to the host.
    """

    if not isinstance(logits, Tensor) or logits.ndim != 2:
        raise ValueError("sampling requires logits with shape [batch, vocabulary]")
    if logits.dtype not in _LOGIT_DTYPES:
        raise ValueError("logits must be float32, float16 or bfloat16")
    if logits.device.type != "cuda":
        raise ValueError("sampling requires CUDA logits")
    rows, vocab = logits.shape
    if not 1 <= vocab <= _MAX_VOCAB:
        raise ValueError("sampling takes 1 to 2^19 columns")
    if not isinstance(uniforms, Tensor) or uniforms.shape != (rows,) or uniforms.dtype != torch.float32 \
            or uniforms.device != logits.device:
        raise ValueError("uniforms must be a float32 [batch] tensor on the logits' device")
    if isinstance(temperature, bool) or not isinstance(temperature, (int, float)) or not 1e-30 <= temperature <= 1e30:
        raise ValueError("temperature must be positive and finite")
    if top_k is not None and (isinstance(top_k, bool) or not isinstance(top_k, int) or top_k < 1):
        raise ValueError("top_k must be a positive integer")
    _check_share("top_p", top_p, False)
    _check_share("min_p", min_p, True)
    if exclude is not None and (isinstance(exclude, bool) or not isinstance(exclude, int) or not 0 <= exclude < vocab):
        raise ValueError("exclude must be an id of the vocabulary")
    z = logits.detach()
    z = z if z.stride(1) == 1 and (rows <= 1 or z.stride(0) >= vocab) else z.contiguous()
    uniforms = uniforms.contiguous()
    ids = torch.empty((rows, 1), device=z.device, dtype=torch.int64)
    probabilities = torch.empty((rows, vocab), device=z.device, dtype=torch.float32) if with_probabilities else None
    need = _workspace_bytes(rows, vocab)
    workspace = torch.empty(need, device=z.device, dtype=torch.uint8) if need else None
    with _native.device_guard(z.device):
        _native.call("koemi_sample_filtered", z.data_ptr(), _native.dtype_code(z.dtype), z.stride(0) if rows > 1 else vocab,
                     rows, vocab, -1 if exclude is None else exclude, float(temperature), min(top_k or 0, 1 << 40),
                     1.0 if top_p is None else float(top_p), 0.0 if min_p is None else float(min_p),
                     uniforms.data_ptr(), ids.data_ptr(), _native.ptr(probabilities), _native.ptr(workspace), need,
                     _native.stream_of(z.device))
    return (ids, probabilities) if with_probabilities else ids


@dataclass(frozen=True)
class SamplingPolicy:
    """Token selection rule applied to one decode step (fast_decode.py:20-37).

    ``temperature`` scales the logits and must be positive. ``top_k`` keeps only
    the highest scoring ids before sampling. ``greedy`` takes the argmax and
    ignores both. The padding id is always removed before selection. ``top_p``
    and ``min_p`` (build-side) restrict further, as in ``sample_tokens``."""

    temperature: float = 1.0
    top_k: int | None = None
    greedy: bool = False
    top_p: float | None = None
    min_p: float | None = None

    def __post_init__(self) -> None:
        if self.temperature <= 0.0:
            raise ValueError("temperature must be positive")
        if self.top_k is not None:
            if isinstance(self.top_k, bool) or not isinstance(self.top_k, int) or self.top_k < 1:
                raise ValueError("top_k must be a positive integer")
        _check_share("top_p", self.top_p, False)
        _check_share("min_p", self.min_p, True)


class TokenSampler:
    """Select decode tokens without reading a tensor value back to the host
    (fast_decode.py:40-95): ``sampler(logits)`` for ``[batch, vocabulary]``
    logits returns ``[batch, 1]`` int64 ids; ``probabilities(logits)`` the
    distribution the policy draws from; ``sample_with_probabilities`` both.
    ``uniforms`` (keyword-only, build-side): ``[batch]`` fp32 numbers in
    [0, 1) to draw with instead of drawing them from ``generator``."""

    def __init__(self, policy: SamplingPolicy, device: torch.device, generator: torch.Generator | None = None) -> None:
        self.policy = policy
        self.device = torch.device(device)
        self.generator = generator

    def _scores(self, logits: Tensor) -> Tensor:
        if logits.ndim != 2:
            raise ValueError("sampling requires logits with shape [batch, vocabulary]")
        if logits.device.type != "cuda":
            raise ValueError("sampling requires CUDA logits")
        scores = logits if logits.dtype == torch.float32 else logits.float()
        return scores if scores.stride(1) == 1 else scores.contiguous()

    def _draw(self, scores: Tensor, probabilities: Tensor | None, uniforms: Tensor | None) -> Tensor:
        batch, vocab = scores.shape
        ids = torch.empty((batch, 1), device=scores.device, dtype=torch.int64)
        if self.policy.greedy:
            _native.call("koemi_herm_greedy_tokens", _native.ptr(scores), scores.stride(0), batch, vocab,
                         PAD_TOKEN_ID, _native.ptr(ids), _native.stream_of(scores.device))
            if probabilities is not None:
                probabilities.zero_().scatter_(-1, ids, 1.0)
            return ids
        if uniforms is None:
            uniforms = torch.rand((batch,), device=scores.device, dtype=torch.float32, generator=self.generator)
        elif uniforms.shape != (batch,) or uniforms.dtype != torch.float32 or uniforms.device != scores.device:
            raise ValueError("uniforms must be a float32 [batch] tensor on the logits' device")
        policy = self.policy
        if policy.top_p is not None or policy.min_p is not None or vocab > _NARROW:
            got = sample_tokens(scores, uniforms, temperature=policy.temperature, top_k=policy.top_k, top_p=policy.top_p,
                                min_p=policy.min_p, exclude=PAD_TOKEN_ID if vocab > PAD_TOKEN_ID else None,
                                with_probabilities=probabilities is not None)
            if probabilities is None:
                return got
            probabilities.copy_(got[1])
            return got[0]
        _native.call("koemi_herm_sample_tokens", _native.ptr(scores), scores.stride(0), batch, vocab, PAD_TOKEN_ID,
                     float(self.policy.temperature), int(self.policy.top_k or 0), _native.ptr(uniforms.contiguous()),
                     _native.ptr(ids), _native.ptr(probabilities), _native.stream_of(scores.device))
        return ids

    def probabilities(self, logits: Tensor) -> Tensor:
        """The distribution this policy draws from, for [batch, vocabulary] logits."""
        return self.sample_with_probabilities(logits)[1]

    def sample_with_probabilities(self, logits: Tensor, *, uniforms: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """[batch, 1] sampled ids together with the distribution they came from."""
        scores = self._scores(logits)
        probabilities = torch.empty(scores.shape, device=scores.device, dtype=torch.float32)
        ids = self._draw(scores, probabilities, uniforms)
        return ids, probabilities

    def __call__(self, logits: Tensor, *, uniforms: Tensor | None = None) -> Tensor:
        """[batch, 1] sampled ids for [batch, vocabulary] logits."""
        return self._draw(self._scores(logits), None, uniforms)
