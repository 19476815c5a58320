"""Low-rank adapters of many requests beside a shared projection (``include/mi_hadamard.h``:
``mi_adapter_plan``, ``mi_lora_add``).

A batch's tokens each name an adapter out of a pool; :func:`adapter_plan` groups them once per batch,
and every projection of every layer uses the plan.  The projection itself is the caller's, for instance
:func:`fp8_gemm_rowscale` on rotated activations.  As elsewhere in the package no autograd graph is
recorded; :func:`lora_add_backward` computes the gradients.  Differentiable inputs are refused under grad mode, in
both directions: there are no second derivatives.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

from . import _lib
from .ops import _DTYPE_CODE, _apart, _dense16, _no_graph, _on_device_of, _require_cuda, _stream, _written

MAX_ADAPTERS, MAX_TOKENS, MAX_RANK, MAX_WIDTH = 1024, 1 << 24, 128, 1 << 22
_LORA = struct.Struct("<4Q4Ii4x")  # mi_lora


class AdapterPlan:
    """A batch's tokens grouped by adapter, on the GPU.

    ``order`` int32 ``[tokens]``: the tokens adapter by adapter, those of one adapter in their own
    order, those without an adapter last.  ``starts`` int32 ``[n_adapters + 1]``: the first position in
    ``order`` of each adapter, and of the tokens without one.
    """

    __slots__ = ("buffer", "tokens", "n_adapters", "_order", "_starts")

    def __init__(self, buffer: torch.Tensor, tokens: int, n_adapters: int, order: int, starts: int):
        self.buffer, self.tokens, self.n_adapters = buffer, tokens, n_adapters
        self._order, self._starts = order, starts

    @property
    def order(self) -> torch.Tensor:
        return self.buffer[self._order:self._order + self.tokens]

    @property
    def starts(self) -> torch.Tensor:
        return self.buffer[self._starts:self._starts + self.n_adapters + 1]


@functools.lru_cache(maxsize=1024)
def _layout(tokens: int, n_adapters: int) -> tuple[int, int, int]:
    out = (ctypes.c_uint64 * 3)()
    _lib.check(_lib.load().mi_adapter_plan_layout(tokens, n_adapters, out), "adapter_plan")
    return tuple(out)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(sizes: bytes, backward: int) -> int:
    return max(_lib.load().mi_lora_workspace(sizes, backward), 16)


def adapter_plan(ids: torch.Tensor, n_adapters: int) -> AdapterPlan:
    """Groups a batch's tokens by adapter: ``ids`` (int32 or int64, ``[tokens]``, on the GPU) names each
    token's adapter in ``[0, n_adapters)``; any other value means none.  No
    synchronisation, so it can be captured with the rest of a step.  The plan serves every
    :func:`lora_add` and :func:`lora_add_backward` on this batch.
    """
    if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"ids must be a vector of int32 or int64 (got {ids.dtype} {tuple(ids.shape)})")
    T = ids.numel()
    if not 1 <= n_adapters <= MAX_ADAPTERS:
        raise RuntimeError(f"n_adapters must be in [1, {MAX_ADAPTERS}], got {n_adapters}")
    if T > MAX_TOKENS:
        raise RuntimeError(f"at most {MAX_TOKENS} tokens, got {T}")
    _require_cuda(ids, "ids")
    lib = _lib.load()
    size, order, starts = _layout(T, n_adapters)
    ids = ids.contiguous()
    buffer = torch.empty(size, dtype=torch.int32, device=ids.device)
    with _on_device_of(ids):
        st = lib.mi_adapter_plan(ids.data_ptr(), 8 * ids.element_size(), T, n_adapters, buffer.data_ptr(), _stream(ids))
    _lib.check(st, "adapter_plan")
    return AdapterPlan(buffer, T, n_adapters, order, starts)


def _row_stride(t: torch.Tensor) -> int:
    """Row stride in elements; one row's stride means nothing."""
    return t.stride(0) if t.size(0) > 1 else 0


def _rows_apart(t: torch.Tensor) -> bool:
    row, column = t.stride()
    return column == 1 and row >= t.size(1) or _apart(t)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _readable(t: torch.Tensor) -> torch.Tensor:
    """``t`` if its rows are contiguous and 16-byte aligned, else a dense copy."""
    if t.numel() == 0 or (t.stride(1) == 1 and t.data_ptr() % 16 == 0 and _row_stride(t) * t.element_size() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check(y, x, A, B, plan, scales, name):
    """Sizes of a call; anything wrong goes to :func:`_refuse`, which says what."""
    dt, dev = x.dtype, x.get_device()
    try:
        (T, K), (Ty, N), (n, r, KA), nNr = x.shape, y.shape, A.shape, B.shape
    except ValueError:
        _refuse(y, x, A, B, plan, scales, name)
    if (dt in _DTYPE_CODE and y.dtype is dt and A.dtype is dt and B.dtype is dt
            and Ty == T and KA == K and nNr == (n, N, r)
            and r % 8 == 0 and 8 <= r <= MAX_RANK and K % 8 == 0 and N % 8 == 0 and 8 <= K <= MAX_WIDTH and 8 <= N <= MAX_WIDTH
            and plan.tokens == T and plan.n_adapters == n
            and dev >= 0 and y.get_device() == dev and A.get_device() == dev and B.get_device() == dev
            and plan.buffer.get_device() == dev
            and (scales is None or (scales.dtype is torch.float32 and scales.shape == (n,) and scales.get_device() == dev))):
        return T, n, r, K, N
    _refuse(y, x, A, B, plan, scales, name)


def _refuse(y, x, A, B, plan, scales, name):
    for t, n, dims in ((y, name, 2), (x, "x", 2), (A, "A", 3), (B, "B", 3)):
        if t.dim() != dims:
            raise RuntimeError(f"{n} must have {dims} dimensions, got {tuple(t.shape)}")
        if t.dtype != x.dtype or t.dtype not in _DTYPE_CODE:
            raise RuntimeError(f"{name}, x, A and B must share a dtype in fp32/bf16/fp16 (got {n} {t.dtype}, x {x.dtype})")
    (T, K), N = x.shape, y.size(1)
    n, r, _ = A.shape
    if y.size(0) != T or A.size(2) != K or tuple(B.shape) != (n, N, r):
        raise RuntimeError(f"shape mismatch: {name} {tuple(y.shape)} x {tuple(x.shape)} A {tuple(A.shape)} B {tuple(B.shape)}")
    if r % 8 or not 8 <= r <= MAX_RANK:
        raise RuntimeError(f"rank must be a multiple of 8 in [8, {MAX_RANK}], got {r}")
    if K % 8 or N % 8 or not (8 <= K <= MAX_WIDTH and 8 <= N <= MAX_WIDTH):
        raise RuntimeError(f"widths must be multiples of 8 in [8, {MAX_WIDTH}], got {K} and {N}")
    if (plan.tokens, plan.n_adapters) != (T, n):
        raise RuntimeError(f"the plan is for {plan.tokens} tokens and {plan.n_adapters} adapters, not {T} and {n}")
    if scales is not None and (scales.dtype != torch.float32 or tuple(scales.shape) != (n,)):
        raise RuntimeError(f"scales must be fp32 [{n}] (got {scales.dtype} {tuple(scales.shape)})")
    _require_cuda(x, "x")
    for t, what in ((y, name), (A, "A"), (B, "B"), (plan.buffer, "plan"), (scales, "scales")):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{what} must be on x's device {x.device}, got {t.device}")
    raise RuntimeError(f"x must be on a GPU (got {x.device})")


def lora_add(y: torch.Tensor, x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, plan: AdapterPlan,
             scales: torch.Tensor | None = None, *, inplace: bool = False, return_shrunk: bool = False):
    """``out[t] = y[t] + scales[a] * B[a] @ (A[a] @ x[t])`` with ``a`` the adapter of token ``t`` in ``plan``;
    ``out[t] = y[t]`` for tokens without one.

    ``y`` ``[tokens, N]`` is the shared projection's output and ``x`` ``[tokens, K]`` its input; ``A``
    ``[n, r, K]`` and ``B`` ``[n, N, r]`` the pool of adapters, all in one dtype (fp32, bf16 or fp16), ranks
    that are multiples of 8 up to 128 (a smaller one is padded with zeros), widths that are multiples of
    8.  ``y`` and ``x`` may be column slices of larger matrices.  ``scales`` fp32 ``[n]``.  Sums are fp32, the
    rank-space vector between the products keeps 23 significand bits or more, and ``out`` is rounded
    once.  ``inplace=True`` writes into ``y`` and returns it.  ``return_shrunk=True`` also returns
    ``A[a] @ x[t]``, fp32 ``[tokens, r]``, which :func:`lora_add_backward` takes.
    """
    _no_graph("lora_add", y, x, A, B, scales)
    T, n, r, K, N = _check(y, x, A, B, plan, scales, "y")
    if inplace and not _rows_apart(y):
        raise RuntimeError("inplace needs a y whose elements do not share memory")
    ys, xs, Ac, Bc = _readable(y), _readable(x), _dense16(A), _dense16(B)
    out = ys if inplace else torch.empty_like(ys, memory_format=torch.contiguous_format)
    shrunk = torch.empty((T, r), dtype=torch.float32, device=x.device) if return_shrunk else None
    if T:
        sc = None if scales is None else scales.contiguous()
        sizes = _LORA.pack(T, _row_stride(xs), _row_stride(ys), _row_stride(out), n, r, K, N, _DTYPE_CODE[x.dtype])
        lib = _lib.load()
        workspace = torch.empty(_workspace_bytes(sizes, 0), dtype=torch.uint8, device=x.device)
        with _on_device_of(x):
            st = lib.mi_lora_add(ys.data_ptr(), xs.data_ptr(), Ac.data_ptr(), Bc.data_ptr(),
                                 _ptr(sc), plan.buffer.data_ptr(), out.data_ptr(),
                                 _ptr(shrunk), workspace.data_ptr(), sizes, _stream(x))
        _lib.check(st, "lora_add")
    if inplace:
        if ys is not y:
            y.copy_(ys)
        else:
            _written(y)
        out = y
    return (out, shrunk) if return_shrunk else out


def lora_add_backward(dy: torch.Tensor, x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, plan: AdapterPlan,
                      scales: torch.Tensor | None = None, *, shrunk: torch.Tensor | None = None,
                      dx: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of :func:`lora_add`: ``(dx, dA, dB)`` from ``dy``, the gradient of ``out`` (the gradient of ``y``
    is ``dy`` itself).  ``shrunk`` is what the forward call returned with ``return_shrunk``; without it
    ``A[a] @ x[t]`` is computed again.  With ``dx`` given (the shared projection's own gradient) the
    adapters' part is added to it in place; without, a new tensor with zeros for tokens without an
    adapter.  ``dA`` and ``dB`` are in the adapters' dtype, zeros for adapters that no token uses; sums
    over tokens are fp32 in a fixed order.
    """
    _no_graph("lora_add_backward", dy, x, A, B, scales, shrunk, dx)
    T, n, r, K, N = _check(dy, x, A, B, plan, scales, "dy")
    dev = x.device
    if shrunk is not None and (shrunk.dtype != torch.float32 or tuple(shrunk.shape) != (T, r) or shrunk.device != dev):
        raise RuntimeError(f"shrunk must be fp32 [{T}, {r}] on {dev} (got {shrunk.dtype} {tuple(shrunk.shape)} on {shrunk.device})")
    if dx is not None:
        if dx.shape != x.shape or dx.dtype != x.dtype or dx.device != dev:
            raise RuntimeError(f"dx must be like x: {tuple(x.shape)} {x.dtype} on {dev}")
        if not _rows_apart(dx):
            raise RuntimeError("dx needs elements that do not share memory")
    gs, xs, Ac, Bc = _readable(dy), _readable(x), _dense16(A), _dense16(B)
    into = torch.empty_like(xs, memory_format=torch.contiguous_format) if dx is None else _readable(dx)
    dA, dB = torch.empty_like(Ac), torch.empty_like(Bc)
    sc = None if scales is None else scales.contiguous()
    u = None if shrunk is None else shrunk.contiguous()
    sizes = _LORA.pack(T, _row_stride(xs), _row_stride(gs), _row_stride(into), n, r, K, N, _DTYPE_CODE[x.dtype])
    lib = _lib.load()
    workspace = torch.empty(_workspace_bytes(sizes, 1), dtype=torch.uint8, device=dev)
    with _on_device_of(x):
        st = lib.mi_lora_add_backward(gs.data_ptr(), xs.data_ptr(), Ac.data_ptr(), Bc.data_ptr(),
                                      _ptr(sc), plan.buffer.data_ptr(),
                                      _ptr(u), None if dx is None else into.data_ptr(),
                                      into.data_ptr(), dA.data_ptr(), dB.data_ptr(), workspace.data_ptr(), sizes, _stream(x))
    _lib.check(st, "lora_add_backward")
    if dx is not None:
        if into is not dx:
            dx.copy_(into)
        else:
            _written(dx)
        into = dx
    return into, dA, dB
