"""Multi-head attention over a window of positions and the first ones (sinks).

The local memory of the reference reads a sliding window with one head as wide as the
model (model/memory.py:332-383). ``window_attention`` is that read with heads, for
prompts and training: position i sees the last ``window`` positions up to its own and the
first ``sinks`` ones, which stay visible. ``WindowCache`` holds what such a window needs of
a sequence in 8 bits, for chunks of a prompt (``window_cache_write``,
``window_cache_entries``) and for single positions (``window_cache_step``,
``window_cache_read``), as the reference's ring does in full (memory.py:385-403). They run
``koemi_window_attention_*`` and ``koemi_window_cache_*``; there is no torch fallback.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from functools import lru_cache
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from koemi_amd import _native
from koemi_amd.think import CudaThinkUnavailableError, CudaThinkValidationError

__all__ = ["WindowCache", "window_attention", "window_cache", "window_cache_entries", "window_cache_read",
           "window_cache_step", "window_cache_write"]

_SUPPORTED_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_MAX_WIDTH = 256
_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}


def _whole(name: str, value: object, least: int) -> int:
    if isinstance(value, bool) or not isinstance(value, int) or value < least:
        raise CudaThinkValidationError(f"{name} must be a {'positive' if least else 'non-negative'} integer")
    return min(value, 1 << 62)


def _scale(scale: object, width: int) -> float:
    if scale is None:
        return 1.0 / math.sqrt(max(width, 1))
    if isinstance(scale, bool) or not isinstance(scale, (int, float)) or not 2.0 ** -126 <= scale < 2.0 ** 127:
        raise CudaThinkValidationError("scale must be a positive finite number")
    return float(scale)


def _load() -> None:
    try:
        _native.load_library()
    except _native.NativeLibraryUnavailableError as error:
        raise CudaThinkUnavailableError(str(error)) from error


def window_attention(queries: Tensor, keys: Tensor, values: Tensor, valid_mask: Tensor | None = None, *, window: int,
                     sinks: int = 0, scale: float | None = None, lengths: Tensor | None = None) -> Tensor:
    """Windowed attention with sinks, with first-order autograd (reverse mode; forward mode is refused).

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

    ``lengths`` ``[B]`` int64, for a chunk behind a cache: ``keys``, ``values`` and ``valid_mask`` are what
    ``window_cache_entries`` gives for these lengths, then the chunk's own (T = sinks + window + L). Rows
    that held fewer than ``sinks`` entries have the others among the chunk's first positions; without ``lengths`` those
    would leave the sight with the window. Without gradients.

    Returns ``[B, L, H, D]`` in the inputs' type. Sums and softmax statistics are float32;
    16-bit calls keep the probabilities and, for the gradients, their derivatives to twice the
    inputs' bits between two products. Sums run in a fixed order. What a value or gradient that is not
    finite reaches is not finite either; an infinity among the gradients may read as NaN there.
    """

    for name, tensor in (("queries", queries), ("keys", keys), ("values", values)):
        if not isinstance(tensor, Tensor):
            raise CudaThinkValidationError(f"{name} must be a torch.Tensor")
    device, dtype = queries.device, queries.dtype
    if keys.device != device or values.device != device or keys.dtype != dtype or values.dtype != dtype:
        raise CudaThinkValidationError("queries, keys and values must share a dtype and a device")
    # asked only while a level is open: each question takes 0.7 us
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (queries, keys, values)):
        raise CudaThinkValidationError("window_attention has no forward-mode derivative")
    trained = torch.is_grad_enabled() and (queries.requires_grad or keys.requires_grad or values.requires_grad)
    window, sinks = _whole("window", window, 1), _whole("sinks", sinks, 0)
    if lengths is not None:
        if not isinstance(lengths, Tensor) or lengths.dtype != torch.int64 or lengths.shape != queries.shape[:1] or lengths.device != device:
            raise CudaThinkValidationError("lengths must be an int64 [batch] tensor on the same device")
        if valid_mask is None or (queries.ndim == keys.ndim == 4 and keys.shape[1] - queries.shape[1] != window + sinks):
            raise CudaThinkValidationError("with lengths, keys, values and a valid_mask must be a cache's sinks + window entries "
                                           "and the queries' own positions")
        if trained:
            raise CudaThinkValidationError("window_attention has no gradients with lengths: a cache's entries have none")
    width = queries.shape[-1] if queries.ndim else 1
    plan = _plan(queries.shape, keys.shape, values.shape, queries.stride(), keys.stride(), values.stride(), dtype, device.type,
                 window, sinks, _scale(scale, width))
    if valid_mask is not None and (not isinstance(valid_mask, Tensor) or valid_mask.dtype != torch.bool
                                   or valid_mask.shape != keys.shape[:2] or valid_mask.device != device):
        raise CudaThinkValidationError("valid_mask must be a bool [batch, total] tensor on the same device")
    if trained:
        return _WindowAttention.apply(queries, keys, values, valid_mask, plan)
    return _forward(queries, keys, values, valid_mask, plan, False, lengths)[0]


class _Plan(NamedTuple):
    """What a call's shapes and numbers come to."""

    sizes: tuple[int, ...]      # batch, length, total, heads, groups, padded width, window, sinks
    width: int                  # of the heads
    scale: float
    code: int                   # of the dtype
    workspace: tuple[int, int]  # bytes, forward and backward
    strides: ctypes.Array | None  # of the inputs as they lie, None where one of them has to be copied


@lru_cache(maxsize=1024)
def _plan(query: tuple, key: tuple, value: tuple, query_stride: tuple, key_stride: tuple, value_stride: tuple,
          dtype: torch.dtype, device: str, window: int, sinks: int, scale: float) -> _Plan:
    """A call's shapes checked, and what follows from them."""

    for name, shape in (("queries", query), ("keys", key), ("values", value)):
        if len(shape) != 4:
            raise CudaThinkValidationError(f"{name} must have shape [batch, length, heads, width]")
    if dtype not in _SUPPORTED_DTYPES:
        raise CudaThinkValidationError("queries, keys and values must be float32, float16 or bfloat16")
    batch, length, heads, width = query
    if key != value or key[0] != batch or key[3] != width:
        raise CudaThinkValidationError("keys and values must have the same shape [batch, total, key heads, width], "
                                       "batch and width being the queries'")
    total, groups = key[1:3]
    if total < length:
        raise CudaThinkValidationError("there must be no fewer keys than queries")
    if heads < 1 or groups < 1 or heads % groups:
        raise CudaThinkValidationError("the key heads must divide the query heads")
    if not 1 <= width <= _MAX_WIDTH:
        raise CudaThinkValidationError(f"heads must be 1 to {_MAX_WIDTH} wide")
    if total * (heads // groups) >= 1 << 29 or batch * groups * -(-max(length * heads // groups, total) // 128) >= 1 << 24:
        raise CudaThinkValidationError("too many positions: 2^29 rows of a key head and 2^24 tiles of 128 rows at most")
    size = dtype.itemsize
    if heads * (width + 8) * size >= 1 << 24:
        raise CudaThinkValidationError("too many heads: a position's must be less than 2^24 bytes")
    if device != "cuda":
        raise CudaThinkValidationError("queries, keys and values must be on CUDA")
    _load()
    padded = -(-width * size // 16) * 16 // size
    code = _native.dtype_code(dtype)
    sizes = (batch, length, total, heads, groups, padded, window, sinks)
    need = (_native.query("koemi_window_attention_workspace_bytes", *sizes, code),
            _native.query("koemi_window_attention_backward_workspace_bytes", *sizes, code))
    strides = (query_stride, key_stride, value_stride)
    in_place = padded == width and all(
        s[3] == 1 and all(x * size % 16 == 0 for x in s[:3]) and s[1] * size < 1 << 24 for s in strides)
    flat = [x for s in strides for x in s[:3]]
    return _Plan(sizes, width, scale, code, need, (ctypes.c_int64 * 9)(*flat) if in_place else None)


def _rows(tensor: Tensor, width: int) -> Tensor:
    """A copy of ``tensor`` [B, L, H, D] that the kernels can read: contiguous whatever the layout, its width
    padded with zeros to whole 16-byte pieces, aligned."""

    batch, length, heads, short = *tensor.shape[:3], width - tensor.shape[3]
    if not short:
        return tensor.clone(memory_format=torch.contiguous_format)
    rows = torch.nn.functional.pad(tensor, (0, short))
    if rows.stride() != (length * heads * width, heads * width, width, 1):  # a layout that pad kept
        rows = tensor.new_zeros((batch, length, heads, width))
        rows[..., :tensor.shape[3]].copy_(tensor)
    return rows


def _strides(*tensors: Tensor) -> ctypes.Array:
    """The batch, position and head strides of [B, L, H, D] tensors, for a host pointer."""

    flat = [s for t in tensors for s in t.stride()[:3]]
    return (ctypes.c_int64 * len(flat))(*flat)


def _forward(queries: Tensor, keys: Tensor, values: Tensor, valid_mask: Tensor | None, plan: _Plan, trained: bool,
             lengths: Tensor | None = None) -> tuple:
    """The output, and with ``trained`` what the gradients need."""

    batch, length, total, heads, groups, padded, window, sinks = plan.sizes
    device = queries.device
    q, k, v, strides = queries, keys, values, plan.strides
    at = (q.data_ptr(), k.data_ptr(), v.data_ptr())
    if strides is None or at[0] % 16 or at[1] % 16 or at[2] % 16:
        q, k, v = (_rows(t.detach(), padded) for t in (q, k, v))
        strides, at = _strides(q, k, v), (q.data_ptr(), k.data_ptr(), v.data_ptr())
    mask = valid_mask.contiguous() if valid_mask is not None else None
    output = torch.empty((batch, length, heads, padded), device=device, dtype=q.dtype)
    rest = torch.empty_like(output) if trained and q.dtype != torch.float32 else None
    lse = torch.empty((batch, heads, length), device=device, dtype=torch.float32) if trained else None
    need = plan.workspace[0]
    workspace = torch.empty(need, device=device, dtype=torch.uint8) if need else None
    if lengths is not None:
        lengths = lengths.contiguous()
        with _native.device_guard(device):
            _native.call("koemi_window_attention_chunk", *at, _native.ptr(mask), strides, lengths.data_ptr(), output.data_ptr(),
                         batch, length, heads, groups, padded, window, sinks, plan.scale, plan.code, _native.ptr(workspace),
                         need, _native.stream_of(device))
        return (output if padded == plan.width else output[..., :plan.width].contiguous(),)
    with _native.device_guard(device):
        _native.call("koemi_window_attention_forward", *at, _native.ptr(mask), strides, output.data_ptr(), _native.ptr(rest),
                     _native.ptr(lse), batch, length, total, heads, groups, padded, window, sinks, plan.scale, plan.code,
                     _native.ptr(workspace), need, _native.stream_of(device))
    result = output if padded == plan.width else output[..., :plan.width].contiguous()
    return (result, q, k, v, mask, output, rest, lse) if trained else (result,)


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(context, queries: Tensor, keys: Tensor, values: Tensor, valid_mask: Tensor | None,  # type: ignore[override]
                plan: _Plan) -> Tensor:
        result, *kept = _forward(queries, keys, values, valid_mask, plan, True)
        context.save_for_backward(*kept)
        context.plan = plan
        return result

    @staticmethod
    @once_differentiable
    def backward(context, d_output: Tensor):  # type: ignore[override]
        q, k, v, mask, output, rest, lse = context.saved_tensors
        plan = context.plan
        batch, length, total, heads, groups, padded, window, sinks = plan.sizes
        device, width = q.device, plan.width
        if padded > width or not d_output.is_contiguous() or d_output.data_ptr() % 16:
            d_output = _rows(d_output, padded)
        d_q, d_k, d_v = (torch.empty(t.shape, device=device, dtype=t.dtype) if need else None
                         for t, need in zip((q, k, v), context.needs_input_grad))
        need = plan.workspace[1]
        workspace = torch.empty(need, device=device, dtype=torch.uint8) if need else None
        with _native.device_guard(device):
            _native.call("koemi_window_attention_backward", q.data_ptr(), k.data_ptr(), v.data_ptr(), _native.ptr(mask),
                         _strides(q, k, v), output.data_ptr(), _native.ptr(rest), lse.data_ptr(), d_output.data_ptr(),
                         _native.ptr(d_q), _native.ptr(d_k), _native.ptr(d_v), batch, length, total, heads, groups, padded,
                         window, sinks, plan.scale, plan.code, _native.ptr(workspace), need, _native.stream_of(device))
        grads = (g if g is None or padded == width else g[..., :width].contiguous() for g in (d_q, d_k, d_v))
        return (*grads, None, None)


@dataclass(frozen=True)
class WindowCache:
    """Keys and values of a window and its sinks, in 8 bits.

    ``keys``, ``values``: codes ``[B, G, window + sinks, stored]``, int8 or float8_e4m3fn,
    ``stored`` being the head width rounded up to 32 (zeros behind it); ``key_scales``,
    ``value_scales`` ``[B, G, window + sinks]`` float32: an entry's row stands for ``codes *
    scale``. Entry p of a row lies at slot p, from ``sinks`` on at ``sinks + (p - sinks) %
    window``. How many entries a row holds is the caller's count, one for all layers. All
    contiguous; ``window_cache`` makes an empty one.
    """

    keys: Tensor
    key_scales: Tensor
    values: Tensor
    value_scales: Tensor
    width: int
    window: int
    sinks: int = 0

    def __post_init__(self) -> None:
        window, sinks = _whole("window", self.window, 1), _whole("sinks", self.sinks, 0)
        width = _whole("width", self.width, 1)
        if width > _MAX_WIDTH:
            raise CudaThinkValidationError(f"heads must be 1 to {_MAX_WIDTH} wide")
        keys, key_scales, values, value_scales = tensors = (self.keys, self.key_scales, self.values, self.value_scales)
        for t in tensors:
            if not isinstance(t, Tensor):
                raise CudaThinkValidationError("a cache is made of four tensors")
        shape, device = keys.shape, keys.device
        if (len(shape) != 4 or shape[2] != window + sinks or shape[3] != -(-width // 32) * 32
                or values.shape != shape or key_scales.shape != shape[:3] or value_scales.shape != shape[:3]):
            raise CudaThinkValidationError("a cache's codes must be [batch, key heads, window + sinks, width rounded up to 32] "
                                           "and its scales [batch, key heads, window + sinks]")
        if keys.dtype not in _CODES or values.dtype != keys.dtype:
            raise CudaThinkValidationError("a cache's codes must be int8 or float8_e4m3fn")
        if key_scales.dtype != torch.float32 or value_scales.dtype != torch.float32:
            raise CudaThinkValidationError("a cache's scales must be float32")
        for t in tensors:
            if t.device != device or not t.is_contiguous():
                raise CudaThinkValidationError("a cache's tensors must be contiguous and on the same device")
        if keys.data_ptr() % 16 or values.data_ptr() % 16:
            raise CudaThinkValidationError("a cache's codes must be 16-byte aligned")

    def buffers(self) -> tuple[int, int, int, int, int]:
        """The entry points' first arguments."""

        return (self.keys.data_ptr(), self.key_scales.data_ptr(), self.values.data_ptr(), self.value_scales.data_ptr(),
                _CODES[self.keys.dtype])


def window_cache(batch: int, heads: int, width: int, *, window: int, sinks: int = 0, dtype: torch.dtype = torch.int8,
                 device: torch.device | str = "cuda") -> WindowCache:
    """An empty cache of ``heads`` key heads of ``width`` for ``batch`` rows (int8 or float8_e4m3fn codes)."""

    batch, heads, width = _whole("batch", batch, 0), _whole("heads", heads, 1), _whole("width", width, 1)
    window, sinks = _whole("window", window, 1), _whole("sinks", sinks, 0)
    if dtype not in _CODES:
        raise CudaThinkValidationError("a cache's codes must be int8 or float8_e4m3fn")
    if width > _MAX_WIDTH:
        raise CudaThinkValidationError(f"heads must be 1 to {_MAX_WIDTH} wide")
    shape = (batch, heads, window + sinks)

    def codes() -> Tensor:
        return torch.zeros((*shape, -(-width // 32) * 32), device=device, dtype=torch.int8).view(dtype)

    return WindowCache(codes(), torch.zeros(shape, device=device), codes(), torch.zeros(shape, device=device),
                       width=width, window=window, sinks=sinks)


def _check_cache(cache: object) -> WindowCache:
    if not isinstance(cache, WindowCache):
        raise CudaThinkValidationError("cache must be a WindowCache")
    return cache


def _check_cuda(cache: WindowCache) -> None:
    if cache.keys.device.type != "cuda":
        raise CudaThinkValidationError("cache must be on CUDA")


def _check_tensor(cache: WindowCache, name: str, tensor: object) -> None:
    if not isinstance(tensor, Tensor):
        raise CudaThinkValidationError(f"{name} must be a torch.Tensor")
    if tensor.device != cache.keys.device:
        raise CudaThinkValidationError(f"{name} must be on the cache's device")


def _check_rows(name: str, shape: tuple[int, ...], wanted: tuple[int, ...], dtype: torch.dtype, same: torch.dtype) -> None:
    """Rows of the cache's heads in one of the three types."""

    if tuple(shape) != wanted:
        raise CudaThinkValidationError(f"{name} must have shape {list(wanted)}")
    if dtype not in _SUPPORTED_DTYPES or dtype != same:
        raise CudaThinkValidationError(f"{name} must be float32, float16 or bfloat16, one type for all")


def _check_counts(cache: WindowCache, name: str, tensor: object) -> Tensor:
    if not isinstance(tensor, Tensor) or tensor.dtype != torch.int64 or tensor.shape != cache.keys.shape[:1] \
            or tensor.device != cache.keys.device:
        raise CudaThinkValidationError(f"{name} must be an int64 [batch] tensor on the cache's device")
    return tensor.contiguous()


def _in_rows(tensor: Tensor) -> Tensor:
    return tensor if tensor.stride(-1) == 1 or tensor.shape[-1] == 1 else tensor.contiguous()


def window_cache_write(cache: WindowCache, keys: Tensor, values: Tensor, lengths: Tensor, counts: Tensor | None = None) -> None:
    """Append rows to the cache, in place.

    ``keys``, ``values`` ``[B, L, G, D]`` (float32, float16 or bfloat16, any strides);
    ``lengths`` ``[B]`` int64: the entries that each row holds already (the caller
    adds what was appended afterwards; a row with a negative one is left as it is);
    ``counts`` ``[B]`` int64: how many of the L each row appends, from the first on (all, when
    omitted; what the others hold does not matter). Of more rows than the ring holds the last
    ones stay. A row's largest absolute value gets the largest code; codes are rounded to
    nearest even; a row that is not finite stands for NaN.
    """

    cache = _check_cache(cache)
    _check_tensor(cache, "keys", keys)
    _check_tensor(cache, "values", values)
    batch, groups = cache.keys.shape[:2]
    length = keys.shape[1] if keys.ndim == 4 else 0
    wanted = (batch, length, groups, cache.width)
    _check_rows("keys", keys.shape, wanted, keys.dtype, keys.dtype)
    _check_rows("values", values.shape, wanted, values.dtype, keys.dtype)
    lengths = _check_counts(cache, "lengths", lengths)
    counts = _check_counts(cache, "counts", counts) if counts is not None else None
    _check_cuda(cache)
    _load()
    k, v = _in_rows(keys.detach()), _in_rows(values.detach())
    with _native.device_guard(k.device):
        _native.call("koemi_window_cache_write", *cache.buffers(), k.data_ptr(), v.data_ptr(), _strides(k, v),
                     lengths.data_ptr(), _native.ptr(counts), batch, length, groups, cache.width, cache.window, cache.sinks,
                     _native.dtype_code(k.dtype), _native.stream_of(k.device))


def window_cache_entries(cache: WindowCache, lengths: Tensor, *, dtype: torch.dtype) -> tuple[Tensor, Tensor, Tensor]:
    """What the cache holds, as the values it stands for.

    Returns ``(keys, values, present)``: ``[B, sinks + window, G, D]`` in ``dtype`` and
    ``[B, sinks + window]`` bool: the sinks, then the last ``window`` other entries in their
    order, the latest at the end; places without an entry hold zeros. Put before the next
    chunk's keys, values and mask, ``window_attention`` with the same ``lengths`` reads them as the
    chunk's own past.
    """

    cache = _check_cache(cache)
    lengths = _check_counts(cache, "lengths", lengths)
    if dtype not in _SUPPORTED_DTYPES:
        raise CudaThinkValidationError("dtype must be float32, float16 or bfloat16")
    _check_cuda(cache)
    _load()
    batch, groups, slots, _ = cache.keys.shape
    device = cache.keys.device
    keys = torch.empty((batch, slots, groups, cache.width), device=device, dtype=dtype)
    values = torch.empty_like(keys)
    present = torch.empty((batch, slots), device=device, dtype=torch.bool)
    with _native.device_guard(device):
        _native.call("koemi_window_cache_entries", *cache.buffers(), lengths.data_ptr(), keys.data_ptr(), values.data_ptr(),
                     present.data_ptr(), batch, groups, cache.width, cache.window, cache.sinks, _native.dtype_code(dtype),
                     _native.stream_of(device))
    return keys, values, present


@lru_cache(maxsize=1024)
def _step_plan(cache: tuple, width: int, window: int, sinks: int, scale: float | None, query: tuple, query_stride: tuple,
               dtype: torch.dtype, key: tuple | None, key_stride: tuple | None, key_dtype: torch.dtype | None,
               value: tuple | None, value_stride: tuple | None, value_dtype: torch.dtype | None) -> tuple:
    """A step's shapes checked: heads, scale, dtype code, bytes of workspace, and the strides of
    the rows as they lie (None where one of them has to be copied)."""

    batch, groups = cache[:2]
    heads = query[1] if len(query) == 3 else 0
    _check_rows("queries", query, (batch, heads, width), dtype, dtype)
    if heads < 1 or heads % groups:
        raise CudaThinkValidationError("the key heads must divide the query heads")
    if key is not None:
        _check_rows("keys", key, (batch, groups, width), key_dtype, dtype)
        _check_rows("values", value, (batch, groups, width), value_dtype, dtype)
    _load()
    need = _native.query("koemi_window_cache_step_workspace_bytes", batch, heads, groups, width, window, sinks)
    strides = (query_stride, key_stride or (0, 0, 1), value_stride or (0, 0, 1))
    flat = (ctypes.c_int64 * 6)(*(x for s in strides for x in s[:2]))
    in_place = width == 1 or all(s[2] == 1 for s in strides)
    return heads, _scale(scale, width), _native.dtype_code(dtype), need, flat if in_place else None


def _step(cache: WindowCache, queries: Tensor, keys: Tensor | None, values: Tensor | None, lengths: Tensor,
          active: Tensor | None, scale: float | None, writes: bool) -> Tensor:
    cache = _check_cache(cache)
    _check_tensor(cache, "queries", queries)
    if scale is not None:
        scale = _scale(scale, cache.width)
    if writes:
        _check_tensor(cache, "keys", keys)
        _check_tensor(cache, "values", values)
    shape, width, window, sinks = cache.keys.shape, cache.width, cache.window, cache.sinks
    new = (keys.shape, keys.stride(), keys.dtype, values.shape, values.stride(), values.dtype) if writes else (None,) * 6
    heads, scale, code, need, strides = _step_plan(shape, width, window, sinks, scale, queries.shape, queries.stride(),
                                                   queries.dtype, *new)
    lengths = _check_counts(cache, "lengths", lengths)
    device = queries.device
    if active is not None:
        if not isinstance(active, Tensor) or active.dtype != torch.bool or active.shape != shape[:1] or active.device != device:
            raise CudaThinkValidationError("active must be a bool [batch] tensor on the cache's device")
        active = active.contiguous()
    _check_cuda(cache)
    q, k, v = queries, keys, values
    if strides is None:
        q, k, v = (_in_rows(t.detach()) if t is not None else None for t in (q, k, v))
        strides = (ctypes.c_int64 * 6)(*(x for t in (q, k, v) for x in (t.stride()[:2] if t is not None else (0, 0))))
    output = torch.empty((shape[0], heads, width), device=device, dtype=q.dtype)
    workspace = torch.empty(need, device=device, dtype=torch.uint8) if need else None
    with _native.device_guard(device):
        _native.call("koemi_window_cache_step", *cache.buffers(), q.data_ptr(), _native.ptr(k), _native.ptr(v), strides,
                     lengths.data_ptr(), _native.ptr(active), output.data_ptr(), shape[0], heads, shape[1], width, window,
                     sinks, scale, code, _native.ptr(workspace), need, _native.stream_of(device))
    return output


def window_cache_step(cache: WindowCache, queries: Tensor, keys: Tensor, values: Tensor, lengths: Tensor,
                      active: Tensor | None = None, *, scale: float | None = None) -> Tensor:
    """One position of every row: its key and value appended, in place, and its queries answered.

    ``queries`` ``[B, H, D]``, ``keys`` and ``values`` ``[B, G, D]`` in one type (float32,
    float16 or bfloat16), G a divisor of H; ``lengths`` ``[B]`` int64: the entries that
    each row holds before the step. Returns ``[B, H, D]``: the softmax read over the sinks
    and the last ``window`` entries, this one among them, as the cache holds them (what
    ``window_attention`` reads at this position, the rounding to 8 bits apart). Rows with
    False in ``active`` ``[B]`` bool, or with a negative length, are left as they are and
    read zeros. Queries and probabilities keep 22 bits or more, sums are float32, in a fixed
    order. Nothing is read back to the host, so a step can be captured in a graph; without
    gradients.
    """

    return _step(cache, queries, keys, values, lengths, active, scale, True)


def window_cache_read(cache: WindowCache, queries: Tensor, lengths: Tensor, active: Tensor | None = None, *,
                      scale: float | None = None) -> Tensor:
    """``window_cache_step`` without a new entry: the queries of the last of ``lengths`` entries."""

    return _step(cache, queries, None, None, lengths, active, scale, False)
