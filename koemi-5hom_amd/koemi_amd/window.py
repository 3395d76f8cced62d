"""Multi-head attention over a window of positions and the first ones (sinks).

The local memory of the reference reads a sliding window with one head as wide as the
model (model/memory.py:332-383). ``window_attention`` is that read with heads, for
prompts and training: position i sees the last ``window`` positions up to its own and the
first ``sinks`` ones, which stay visible. It runs ``koemi_window_attention_forward`` and
``koemi_window_attention_backward``; there is no torch fallback.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from koemi_amd import _native
from koemi_amd.think import CudaThinkUnavailableError, CudaThinkValidationError

__all__ = ["window_attention"]

_SUPPORTED_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_MAX_WIDTH = 256


def _whole(name: str, value: object, least: int) -> int:
    if isinstance(value, bool) or not isinstance(value, int) or value < least:
        raise CudaThinkValidationError(f"{name} must be a {'positive' if least else 'non-negative'} integer")
    return min(value, 1 << 62)


def _scale(scale: object, width: int) -> float:
    if scale is None:
        return 1.0 / math.sqrt(width)
    if isinstance(scale, bool) or not isinstance(scale, (int, float)) or not 2.0 ** -126 <= scale < 2.0 ** 127:
        raise CudaThinkValidationError("scale must be a positive finite number")
    return float(scale)


def _load() -> None:
    try:
        _native.load_library()
    except _native.NativeLibraryUnavailableError as error:
        raise CudaThinkUnavailableError(str(error)) from error


def window_attention(queries: Tensor, keys: Tensor, values: Tensor, valid_mask: Tensor | None = None, *, window: int,
                     sinks: int = 0, scale: float | None = None) -> Tensor:
    """Windowed attention with sinks, with first-order autograd.

    ``queries`` ``[B, L, H, D]``, ``keys`` and ``values`` ``[B, T, G, D]`` in one type
    (float32, float16 or bfloat16), D at most 256, G a divisor of H (query head h reads
    key head ``h // (H / G)``), T at least L: the queries stand at the last L of the T
    positions, so keys carried from earlier chunks come first. Any strides; rows with
    contiguous columns are read in place.

    Query i reads ``sum_j softmax_j(scale q_i . k_j) v_j`` over the positions j <= i with
    ``i - j < window`` or ``j < sinks``; ``scale`` is 1 / sqrt(D) unless given.
    ``valid_mask`` ``[B, T]`` bool: a masked position takes no part, as key or as query; what
    its tensors hold does not matter, it reads zeros and its gradients are zeros. A query
    that sees nothing reads zeros. Positions count from the first row of ``keys``, so
    batches are padded at their end.

    Returns ``[B, L, H, D]`` in the inputs' type. Sums and softmax statistics are float32;
    16-bit calls round the probabilities (and, for the gradients, their derivatives) to the
    inputs' type between two products. Sums run in a fixed order.
    """

    tensors = {"queries": queries, "keys": keys, "values": values}
    for name, tensor in tensors.items():
        if not isinstance(tensor, Tensor):
            raise CudaThinkValidationError(f"{name} must be a torch.Tensor")
        if tensor.ndim != 4:
            raise CudaThinkValidationError(f"{name} must have shape [batch, length, heads, width]")
        if tensor.dtype not in _SUPPORTED_DTYPES:
            raise CudaThinkValidationError(f"{name} must be float32, float16 or bfloat16")
        if tensor.device.type != "cuda":
            raise CudaThinkValidationError(f"{name} must be on CUDA")
    if len({t.device for t in tensors.values()}) != 1 or len({t.dtype for t in tensors.values()}) != 1:
        raise CudaThinkValidationError("queries, keys and values must share a dtype and a device")
    batch, length, heads, width = queries.shape
    if keys.shape != values.shape or keys.shape[0] != batch or keys.shape[3] != width:
        raise CudaThinkValidationError("keys and values must have the same shape [batch, total, key heads, width], "
                                       "batch and width being the queries'")
    total, groups = keys.shape[1:3]
    if total < length:
        raise CudaThinkValidationError("there must be no fewer keys than queries")
    if heads < 1 or groups < 1 or heads % groups:
        raise CudaThinkValidationError("the key heads must divide the query heads")
    if not 1 <= width <= _MAX_WIDTH:
        raise CudaThinkValidationError(f"heads must be 1 to {_MAX_WIDTH} wide")
    if total * (heads // groups) >= 1 << 29 or batch * groups * -(-max(length * heads // groups, total) // 128) >= 1 << 24:
        raise CudaThinkValidationError("too many positions: 2^29 rows of a key head and 2^24 tiles of 128 rows at most")
    if valid_mask is not None and (not isinstance(valid_mask, Tensor) or valid_mask.dtype != torch.bool
                                   or valid_mask.shape != (batch, total) or valid_mask.device != queries.device):
        raise CudaThinkValidationError("valid_mask must be a bool [batch, total] tensor on the same device")
    window, sinks, scale = _whole("window", window, 1), _whole("sinks", sinks, 0), _scale(scale, width)
    _load()
    trained = torch.is_grad_enabled() and any(t.requires_grad for t in tensors.values())
    return _WindowAttention.apply(queries, keys, values, valid_mask, window, sinks, scale, trained)


@lru_cache(maxsize=256)
def _workspace_bytes(batch: int, length: int, total: int, heads: int, groups: int, width: int, window: int, sinks: int,
                     dtype: int) -> tuple[int, int]:
    """Bytes of workspace of a shape: forward, backward."""

    shape = (batch, length, total, heads, groups, width, window, sinks, dtype)
    return (_native.query("koemi_window_attention_workspace_bytes", *shape),
            _native.query("koemi_window_attention_backward_workspace_bytes", *shape))


def _strides(*tensors: Tensor) -> ctypes.Array:
    """The batch, position and head strides of [B, L, H, D] tensors, for a host pointer."""

    flat = [s for t in tensors for s in t.stride()[:3]]
    return (ctypes.c_int64 * len(flat))(*flat)


def _bytes(need: int, device: torch.device) -> Tensor | None:
    return torch.empty(need, device=device, dtype=torch.uint8) if need else None


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(context, queries: Tensor, keys: Tensor, values: Tensor, valid_mask: Tensor | None,  # type: ignore[override]
                window: int, sinks: int, scale: float, trained: bool) -> Tensor:
        batch, length, heads, width = queries.shape
        total, groups = keys.shape[1:3]
        device, code = queries.device, _native.dtype_code(queries.dtype)
        q, k, v = (t if t.stride(3) == 1 or width == 1 else t.contiguous() for t in (queries, keys, values))
        mask = valid_mask.contiguous() if valid_mask is not None else None
        output = torch.empty((batch, length, heads, width), device=device, dtype=queries.dtype)
        rest = torch.empty_like(output) if trained and queries.dtype != torch.float32 else None
        lse = torch.empty((batch, heads, length), device=device, dtype=torch.float32) if trained else None
        shape = (batch, length, total, heads, groups, width, window, sinks)
        need = _workspace_bytes(*shape, code)[0]
        workspace = _bytes(need, device)
        with _native.device_guard(device):
            _native.call("koemi_window_attention_forward", q.data_ptr(), k.data_ptr(), v.data_ptr(), _native.ptr(mask),
                         _strides(q, k, v), output.data_ptr(), _native.ptr(rest), _native.ptr(lse), *shape, scale, code,
                         _native.ptr(workspace), need, _native.stream_of(device))
        if trained:
            context.save_for_backward(q, k, v, mask, output, rest, lse)
            context.window = (window, sinks, scale)
        return output

    @staticmethod
    @once_differentiable
    def backward(context, d_output: Tensor):  # type: ignore[override]
        q, k, v, mask, output, rest, lse = context.saved_tensors
        window, sinks, scale = context.window
        batch, length, heads, width = q.shape
        total, groups = k.shape[1:3]
        device, code = q.device, _native.dtype_code(q.dtype)
        d_output = d_output.contiguous()
        wanted = context.needs_input_grad
        d_q, d_k, d_v = (torch.empty(t.shape, device=device, dtype=t.dtype) if need else None
                         for t, need in zip((q, k, v), wanted))
        shape = (batch, length, total, heads, groups, width, window, sinks)
        need = _workspace_bytes(*shape, code)[1]
        workspace = _bytes(need, device)
        with _native.device_guard(device):
            _native.call("koemi_window_attention_backward", q.data_ptr(), k.data_ptr(), v.data_ptr(), _native.ptr(mask),
                         _strides(q, k, v), output.data_ptr(), _native.ptr(rest), lse.data_ptr(), d_output.data_ptr(),
                         _native.ptr(d_q), _native.ptr(d_k), _native.ptr(d_v), *shape, scale, code,
                         _native.ptr(workspace), need, _native.stream_of(device))
        return d_q, d_k, d_v, None, None, None, None, None
