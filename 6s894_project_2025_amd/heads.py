"""Query and key heads between a projection and attention: per-head RMS norm, position rotation and
the Hadamard rotation of the head in one pass (``include/mi_hadamard.h``: ``mi_qk_norm_rope``).

Like the other ops of the package these record no autograd graph: the gradients are a function of
their own, and a differentiable input under an active grad mode is an error rather than a silent
detach (call them under ``torch.no_grad()`` or inside a ``torch.autograd.Function``; the gradient
function has no derivative of its own, so such a Function's backward pass is ``once_differentiable``).
"""
from __future__ import annotations

import struct

import torch

from . import _lib
from .ops import _DTYPE_CODE, _apart, _dense16, _is_pow2, _no_graph, _on_device_of, _require_cuda, _stream, _written

_NEIGHBOURS, _HADAMARD = 1, 2
_HEADS = struct.Struct("<Q6Q6Q4I" "I4I" "iiIII" "f4x")  # mi_heads
_MAX_D = 512


def _readable(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """``t`` as the kernels address it (heads contiguous, 16-byte aligned base and strides), a dense copy if it is
    not, with its token and head stride in elements; 0 along an axis of one entry, whose stride means nothing."""
    T, H, D = t.shape
    ts, hs, ds = t.stride()
    if T <= 1:
        ts = 0
    if H <= 1:
        hs = 0
    align = 15 // t.element_size()  # a power of two less one
    if ds == 1 and not (ts | hs) & align and t.data_ptr() % 16 == 0 or T * H == 0:
        return t, ts, hs
    return t.clone(memory_format=torch.contiguous_format), H * D, D


def _describe(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, interleaved, hadamard):
    """The operands that both directions share: (tokens, heads, D and the rest of mi_heads behind the strides).
    Anything wrong goes to :func:`_refuse`, which says what."""
    dt, dev = q.dtype, q.get_device()
    try:
        (T, Hq, D), (Tk, Hk, Dk), (half,), pshape = q.shape, k.shape, inv_freq.shape, positions.shape
    except ValueError:
        _refuse(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, hadamard)
    axes = 1 if len(pshape) == 1 else pshape[0] if len(pshape) == 2 else 0
    if sections is None:
        ends = (half, 0, 0, 0)
        fits = axes == 1
    else:
        ends, total = [], 0
        for s in sections:
            total += int(s)
            ends.append(total)
        fits = 1 <= len(ends) == axes <= 4 and total == half and min(sections) >= 0
        ends += [0] * (4 - axes)
    weights = [w for w in (q_weight, k_weight) if w is not None]
    wdt = weights[0].dtype if weights else dt
    if not (fits and dt in _DTYPE_CODE and k.dtype is dt and Tk == T and Dk == D and D % 16 == 0 and 16 <= D <= _MAX_D
            and eps >= 0.0 and half % 8 == 0 and 2 * half <= D and pshape[-1] == T
            and (positions.dtype is torch.int32 or positions.dtype is torch.int64)
            and (inv_freq.dtype is torch.float32 or inv_freq.dtype is torch.float64)
            and (wdt is dt or wdt is torch.float32) and not (hadamard and not _is_pow2(D))
            and all(w.shape == (D,) and w.dtype is wdt and w.get_device() == dev for w in weights)
            and dev >= 0 and k.get_device() == dev and positions.get_device() == dev and inv_freq.get_device() == dev):
        _refuse(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, hadamard)
    flags = (_NEIGHBOURS if interleaved else 0) | (_HADAMARD if hadamard else 0)
    return T, D, wdt, (Hq, Hk, D, 2 * half, axes, *ends, _DTYPE_CODE[dt], _DTYPE_CODE[wdt], 8 * positions.element_size(),
                       8 * inv_freq.element_size(), flags, eps)


def _refuse(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, hadamard):
    for t, n in ((q, "q"), (k, "k")):
        if t.dim() != 3:
            raise RuntimeError(f"{n} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    if q.dtype not in _DTYPE_CODE or k.dtype != q.dtype:
        raise RuntimeError(f"q and k must share a dtype in fp32/bf16/fp16 (got {q.dtype}, {k.dtype})")
    T, _, D = q.shape
    if k.size(0) != T or k.size(2) != D:
        raise RuntimeError(f"shape mismatch: q {tuple(q.shape)} k {tuple(k.shape)}")
    if D % 16 or not 16 <= D <= _MAX_D:
        raise RuntimeError(f"head_dim must be a multiple of 16 in [16, {_MAX_D}], got {D}")
    if hadamard and not _is_pow2(D):
        raise RuntimeError(f"hadamard needs a power-of-two head_dim, got {D}")
    if not eps >= 0.0:
        raise RuntimeError(f"eps must not be negative, got {eps}")
    if inv_freq.dim() != 1 or inv_freq.dtype not in (torch.float32, torch.float64):
        raise RuntimeError("inv_freq must be a vector in fp32 or fp64")
    half = inv_freq.numel()
    if half % 8 or 2 * half > D:
        raise RuntimeError(f"inv_freq must hold a multiple of 8 frequencies, at most head_dim / 2 = {D // 2}, got {half}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"positions must be int32 or int64 (got {positions.dtype})")
    axes = 1 if positions.dim() == 1 else positions.size(0)
    if positions.dim() not in (1, 2) or positions.size(-1) != T or not 1 <= axes <= 4:
        raise RuntimeError(f"positions must be [tokens] or [axes, tokens] with up to four axes, got "
                           f"{tuple(positions.shape)} for {T} tokens")
    if sections is None:
        if axes != 1:
            raise RuntimeError("positions with several axes need sections")
    else:
        ends, total = [], 0
        for s in sections:
            if s < 0:
                raise RuntimeError(f"sections must not be negative, got {tuple(sections)}")
            total += int(s)
            ends.append(total)
        if len(ends) != axes or total != half:
            raise RuntimeError(f"sections {tuple(sections)} must give each of the {axes} axes its share of the {half} frequencies")
    kinds = set()
    for w, n in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is None:
            continue
        if w.dim() != 1 or w.numel() != D:
            raise RuntimeError(f"{n} must have {D} entries")
        if w.dtype not in (q.dtype, torch.float32):
            raise RuntimeError(f"{n} must be in the heads' dtype or fp32 (got {w.dtype})")
        kinds.add(w.dtype)
    if len(kinds) > 1:
        raise RuntimeError("q_weight and k_weight must share a dtype")
    _require_cuda(q, "q")
    for t, n in ((k, "k"), (q_weight, "q_weight"), (k_weight, "k_weight"), (positions, "positions"),
                 (inv_freq, "inv_freq")):
        if t is not None and t.device != q.device:
            raise RuntimeError(f"{n} must be on q's device {q.device}, got {t.device}")
    raise RuntimeError("unsupported operands")


def _ptr(t):
    return None if t is None else t.data_ptr()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 positions: torch.Tensor, inv_freq: torch.Tensor, *, eps: float = 1e-6,
                 sections=None, interleaved: bool = False, hadamard: bool = False,
                 inplace: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each query and key head, rotation by the token's position and, with ``hadamard``,
    ``H_D / sqrt(D)`` over the head, in one kernel; returns ``(q_out, k_out)``.

    ``q`` ``[tokens, q_heads, D]`` and ``k`` ``[tokens, k_heads, D]`` in fp32, bf16 or fp16 may be views
    into one packed projection output; ``D`` is a multiple of 16 up to 512.  Weights ``[D]`` (the heads'
    dtype or fp32; ``None`` for ones).  Pair ``f`` turns by ``position * inv_freq[f]`` radians:
    ``inv_freq`` (fp32 or fp64, a multiple of 8 frequencies) sets the rotary width ``R = 2 * len``, and
    the values from ``R`` on are only normed.  The pairs are ``(i, i + R/2)``, or ``(2i, 2i + 1)`` with
    ``interleaved``.  ``positions`` is ``[tokens]``, or ``[axes, tokens]`` with ``sections`` counting the
    consecutive frequencies of each axis (time, height, width, ...).  Angles are formed in fp64, so far
    positions keep their accuracy; the rest is fp32 with one rounding at the end.
    ``inplace=True`` writes into ``q`` and ``k`` and returns them.
    """
    _no_graph("qk_norm_rope", q, k, q_weight, k_weight, inv_freq)
    T, D, _, rest = _describe(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, interleaved, hadamard)
    if inplace and not _apart(q, k):
        raise RuntimeError("inplace needs q and k whose elements do not share memory")
    (qs, qt, qh), (ks, kt, kh) = _readable(q), _readable(k)
    if inplace:
        qo, ko, qot, qoh, kot, koh = qs, ks, qt, qh, kt, kh
    else:
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
        qot, qoh, kot, koh = rest[0] * D, D, rest[1] * D, D
    if qo.numel() or ko.numel():
        qw = None if q_weight is None else _dense16(q_weight)
        kw = None if k_weight is None else _dense16(k_weight)
        pos, freq = positions.contiguous(), inv_freq.contiguous()
        lib = _lib.load()
        with _on_device_of(q):
            st = lib.mi_qk_norm_rope(qs.data_ptr(), ks.data_ptr(), _ptr(qw), _ptr(kw), pos.data_ptr(), freq.data_ptr(), qo.data_ptr(),
                                     ko.data_ptr(), _HEADS.pack(T, qt, kt, qot, kot, 0, 0, qh, kh, qoh, koh, 0, 0, *rest), _stream(q))
        _lib.check(st, "qk_norm_rope")
    if inplace:
        for given, written in ((q, qs), (k, ks)):
            if written is not given:
                given.copy_(written)
            else:
                _written(given)
        return q, k
    return qo, ko


def qk_norm_rope_backward(q_grad: torch.Tensor, k_grad: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                          q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                          positions: torch.Tensor, inv_freq: torch.Tensor, *, eps: float = 1e-6,
                          sections=None, interleaved: bool = False, hadamard: bool = False):
    """Gradients of :func:`qk_norm_rope`: ``(dq, dk, dq_weight, dk_weight)`` from the gradients of its
    outputs and its inputs ``q``, ``k`` (before the call, so not from an in-place one).  A weight that is
    ``None`` has gradient ``None``; the others are in the weights' dtype, summed over all tokens and
    heads in fp32 in a fixed order.
    """
    _no_graph("qk_norm_rope_backward", q_grad, k_grad, q, k, q_weight, k_weight, inv_freq)
    T, D, wdt, rest = _describe(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, interleaved, hadamard)
    for g, t, n in ((q_grad, q, "q_grad"), (k_grad, k, "k_grad")):
        if g.shape != t.shape or g.dtype is not t.dtype:
            raise RuntimeError(f"{n} must have the shape and dtype of {n[0]}: {tuple(t.shape)} {t.dtype}, got "
                               f"{tuple(g.shape)} {g.dtype}")
        if g.device != t.device:
            raise RuntimeError(f"{n} must be on q's device {q.device}, got {g.device}")
    dev = q.device
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dqw = None if q_weight is None else torch.empty(D, dtype=wdt, device=dev)
    dkw = None if k_weight is None else torch.empty(D, dtype=wdt, device=dev)
    (qs, qt, qh), (ks, kt, kh), (qg, qgt, qgh), (kg, kgt, kgh) = _readable(q), _readable(k), _readable(q_grad), _readable(k_grad)
    qw = None if q_weight is None else _dense16(q_weight)
    kw = None if k_weight is None else _dense16(k_weight)
    pos, freq = positions.contiguous(), inv_freq.contiguous()
    lib = _lib.load()
    workspace = None
    if dqw is not None or dkw is not None:
        workspace = torch.empty(lib.mi_qk_norm_rope_workspace(T, D), dtype=torch.uint8, device=dev)
    with _on_device_of(q):
        st = lib.mi_qk_norm_rope_backward(qs.data_ptr(), ks.data_ptr(), qg.data_ptr(), kg.data_ptr(), _ptr(qw), _ptr(kw),
                                          pos.data_ptr(), freq.data_ptr(), dq.data_ptr(), dk.data_ptr(), _ptr(dqw), _ptr(dkw),
                                          _ptr(workspace),
                                          _HEADS.pack(T, qt, kt, qgt, kgt, rest[0] * D, rest[1] * D, qh, kh, qgh, kgh, D, D, *rest),
                                          _stream(q))
    _lib.check(st, "qk_norm_rope_backward")
    return dq, dk, dqw, dkw
