"""Rotary positions of one axis on the HIP kernels: interleaved and half layouts, part of a head, frequencies scaled for
contexts longer than the trained one; and the norm of each head's queries and keys in the same pass.

Beside `producer.axial_rope` (AxialRoPE, streamvoxel/models/unconditional_md4.py:10-24), which turns the three axes of
the reference's positions with the reference's bf16 roundings; no counterpart in the reference.
"""
from __future__ import annotations

import math
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from streamvoxel_amd import _lib

__all__ = ['rotary', 'rotary_frequencies', 'norm_rotary']

LAYOUTS = {'half': _lib.SVHIP_ROTARY_HALF, 'interleaved': _lib.SVHIP_ROTARY_INTERLEAVED}


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None, low=1.0, high=32.0,
                       device=None):
    """(frequencies, amplitude): the fp64 frequencies base^(-2i / rotary_dim), i < rotary_dim / 2, in radians a
    position, and the factor of the turned pairs, 1 unless the scaling changes it. `scaling` for contexts `factor`
    times as long as the trained one:
      'linear': every frequency divided by `factor` (position interpolation);
      'wavelength': the pairs that make fewer than `low` turns over `original_length` trained positions divided by it,
        those that make more than `high` kept, a linear ramp in between, and the amplitude 0.1 ln(factor) + 1 (the
        by-parts interpolation of "YaRN: Efficient Context Window Extension of Large Language Models")."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError('rotary_dim must be positive and even')
    if scaling not in (None, 'linear', 'wavelength'):
        raise ValueError("scaling is None, 'linear' or 'wavelength'")
    if not factor >= 1.0:
        raise ValueError('factor must be at least 1')
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    amplitude = 1.0
    if scaling == 'linear':
        freq = freq / factor
    elif scaling == 'wavelength':
        if not original_length or not low < high:
            raise ValueError("'wavelength' needs original_length, and low below high")
        turns = original_length * freq / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
        amplitude = 0.1 * math.log(factor) + 1.0
    return (freq if device is None else freq.to(device)), amplitude


_ARGS = struct.Struct('4P17qd')   # svhip_rotary_args


def _launch(x, out, positions, frequencies, layout, amplitude, inverse):
    args = _ARGS.pack(x.data_ptr(), out.data_ptr(), positions.data_ptr(), frequencies.data_ptr(),
                      _lib.dtype_code(x.dtype), positions.dtype == torch.int64, frequencies.numel(), LAYOUTS[layout],
                      inverse, *x.shape, *x.stride()[:3], *out.stride()[:3],
                      positions.stride(0) if positions.dim() == 2 else 0, positions.stride(-1), amplitude)
    _lib.launch('svhip_rotary', x, args)
    return out


def _tracked(x):
    """True where a gradient or a tangent goes through x."""
    if torch.is_grad_enabled() and x.requires_grad:
        return True
    # (The level first: a look for the tangent takes 1.8 us.)
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None


def _turn(x, positions, frequencies, layout, amplitude, inverse):
    x = x if x.stride(-1) == 1 else x.contiguous()
    if _tracked(x):
        return _Rotary.apply(x, positions, frequencies, layout, amplitude, inverse)
    return _launch(x, _lib.rows_like(x), positions, frequencies, layout, amplitude, inverse)


class _Rotary(torch.autograd.Function):
    """The rotation, or its transpose (inverse 1): linear, so that each is the other's gradient, as often as asked for,
    and a tangent turns as x does."""

    @staticmethod
    def forward(ctx, x, positions, frequencies, layout, amplitude, inverse):
        ctx.save_for_backward(positions, frequencies)
        ctx.save_for_forward(positions, frequencies)
        ctx.args = layout, amplitude, inverse
        return _launch(x, _lib.rows_like(x), positions, frequencies, layout, amplitude, inverse)

    @staticmethod
    def backward(ctx, dy):
        layout, amplitude, inverse = ctx.args
        return _turn(dy, *ctx.saved_tensors, layout, amplitude, 1 - inverse), None, None, None, None, None

    @staticmethod
    def jvp(ctx, dx, *_):
        return _turn(dx, *ctx.saved_tensors, *ctx.args)


def rotary(x, positions, frequencies, layout='half', amplitude=1.0, out=None):
    """Rotary positions of x [B,H,N,D] bf16 or fp32 (head_dim contiguous, any other strides; packed tokens as
    [1,H,T,D]) at integer positions [N] or [B,N] (int32 or int64, any sign): pair i of the first 2 * len(frequencies)
    elements turns by positions * frequencies[i] and is scaled by `amplitude`, the other elements are kept. `layout`
    'half' pairs element i with i + len(frequencies), 'interleaved' 2i with 2i + 1. frequencies: the fp64 buffer of
    `rotary_frequencies`, at most 128 pairs. The turns are formed in 64 bits (far positions keep their angle), the
    rest in fp32, rounded once to x's type. Differentiable in x, backwards and forwards (captured into a graph: for
    leaves that no eager graph still holds). `out` (optional, no gradient or tangent through it; x itself, or memory
    that x does not share) receives the result; returns it."""
    _lib.require_one_gpu(x, positions, frequencies, out)
    if layout not in LAYOUTS:
        raise ValueError("layout is 'half' or 'interleaved'")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError('x must be bfloat16 or float32')
    if x.dim() != 4 or x.stride(-1) != 1:
        raise ValueError('x must be [B, H, N, D] with a contiguous head_dim')
    B, H, N, D = x.shape
    if positions.dtype not in (torch.int32, torch.int64) or (positions.shape != (N,) and positions.shape != (B, N)):
        raise ValueError(f'positions must be int32 or int64 [N] or [B, N], got {positions.dtype} {tuple(positions.shape)}')
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous():
        raise ValueError('frequencies must be a contiguous fp64 vector')
    if not 1 <= frequencies.numel() <= min(D // 2, 128):
        raise ValueError(f'{frequencies.numel()} frequencies do not fit head_dim {D} (at most 128)')
    if out is None:
        if _tracked(x):
            return _Rotary.apply(x, positions, frequencies, layout, float(amplitude), 0)
        out = _lib.rows_like(x)
    else:
        if _tracked(x) or _tracked(out):
            raise ValueError('out= takes no part in a gradient')
        if out.shape != x.shape or out.dtype != x.dtype or out.stride(-1) != 1 or _lib.stacked(out):
            raise ValueError("out must have x's shape and type, a contiguous head_dim and a place for every element")
        if _lib.overlaps(x, out) and (x.data_ptr() != out.data_ptr() or x.stride() != out.stride()):
            raise ValueError('out must be x itself or memory that x does not share')
        if _lib.overlaps_any(out, positions, frequencies):
            raise ValueError('out must not share memory with positions or frequencies')
    return _launch(x, out, positions, frequencies, layout, float(amplitude), 0)


_NORM = struct.Struct('13P31q2d')   # svhip_norm_rotary_args


_NONE = 0, 0, 0
_DTYPES = {torch.float32: _lib.SVHIP_F32, torch.bfloat16: _lib.SVHIP_BF16}
_WHOLE = torch.int32, torch.int64


def _places(t):
    return _NONE if t is None else t.stride()[:3]


def _address(t):
    return 0 if t is None else t.data_ptr()


def _norm_args(query, key, dq, dk, weights, outs, dw, workspace, positions, frequencies, dtype, weight_dtype, layout, amplitude,
               eps):
    """The svhip_norm_rotary_args of a gradient."""
    B, H, N, D = query.shape
    return _NORM.pack(_address(query), _address(key), _address(dq), _address(dk), *map(_address, weights), *map(_address, outs),
                      *map(_address, dw), positions.data_ptr(), frequencies.data_ptr(), _address(workspace),
                      0 if workspace is None else workspace.numel(), dtype, weight_dtype, positions.dtype == torch.int64,
                      frequencies.numel(), layout, B, H, 0 if key is None else key.shape[1], N, D, *_places(query),
                      *_places(key), *_places(dq), *_places(dk), *_places(outs[0]), *_places(outs[1]),
                      positions.stride(0) if positions.dim() == 2 else 0, positions.stride(-1), amplitude, eps)


def _normed(query, key, wq, wk, outs, positions, frequencies, dtype, weight_dtype, layout, amplitude, eps):
    # (Packed here: half of _norm_args' time.)
    B, H, N, D = query.shape
    q, k = outs
    Hk, ka, sk, ko, so = 0, 0, _NONE, 0, _NONE
    if key is not None:
        Hk, ka, sk, ko, so = key.shape[1], key.data_ptr(), key.stride()[:3], k.data_ptr(), k.stride()[:3]
    sp = positions.stride()
    args = _NORM.pack(query.data_ptr(), ka, 0, 0, 0 if wq is None else wq.data_ptr(), 0 if wk is None else wk.data_ptr(),
                      q.data_ptr(), ko, 0, 0, positions.data_ptr(), frequencies.data_ptr(), 0, 0, dtype, weight_dtype,
                      positions.dtype == torch.int64, frequencies.numel(), layout, B, H, Hk, N, D, *query.stride()[:3], *sk,
                      *_NONE, *_NONE, *q.stride()[:3], *so, sp[0] if len(sp) == 2 else 0, sp[-1], amplitude, eps)
    _lib.launch('svhip_norm_rotary', query, args)
    return outs


def _like(t):
    return None if t is None else _lib.rows_like(t)


def _rows(t):
    """Rows with a contiguous head_dim: the tensor itself, or a copy."""
    return t if t is None or t.stride(-1) == 1 else t.contiguous()


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, *how):
        positions, frequencies, *rest = how
        ctx.save_for_backward(query, key, query_weight, key_weight, positions, frequencies)
        ctx.rest = rest
        q, k = _normed(query, key, query_weight, key_weight, (_like(query), _like(key)), *how)
        return q if k is None else (q, k)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        query, key, *weights, positions, frequencies = ctx.saved_tensors
        dq, dk = _rows(dq), _rows(dk)
        needs = ctx.needs_input_grad
        outs = [_lib.rows_like(t) if need else None for t, need in zip((query, key), needs)]
        dw = [torch.empty_like(t) if need else None for t, need in zip(weights, needs[2:])]
        B, H, N, D = query.shape
        workspace = None
        if dw[0] is not None or dw[1] is not None:
            nbytes = _lib.load().svhip_norm_rotary_workspace_bytes(B, H, 0 if key is None else key.shape[1], N, D)
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
        _lib.launch('svhip_norm_rotary_grad', query, _norm_args(query, key, dq, dk, weights, outs, dw, workspace, positions,
                                                                frequencies, *ctx.rest))
        return *outs, *dw, *[None] * (2 + len(ctx.rest))


def norm_rotary(query, key, query_weight, key_weight, positions, frequencies, eps=1e-6, layout='half', amplitude=1.0, out=None):
    """(query, key) normed for each head and turned by their rotary positions, in one pass: a row x becomes
    x / sqrt(mean(x^2) + eps) * weight, and then what `rotary` makes of it.

    query [B,H,N,D] and key [B,Hk,N,D] (or None: the queries alone, key_weight None too; the second result is None then),
    both bf16 or fp32, head_dim contiguous with any other strides, 2 <= D <= 256; query_weight and key_weight [D], fp32 or
    bf16 alike, one for all heads, or None for ones. positions, frequencies, layout and amplitude as `rotary` takes them.
    fp32 throughout (a row's squares must not pass its range), rounded once to the rows' type. Differentiable in the rows
    and the weights, once and backwards; the weights' gradients are the same bits from call to call. Captured into a graph:
    for leaves that no eager graph still holds. `out` (optional, no gradient through it): the pair that receives the
    results, each its input itself or memory that neither input shares."""
    _lib.require_one_gpu(query, key, query_weight, key_weight, positions, frequencies, *(out or ()))
    if layout not in LAYOUTS:
        raise ValueError("layout is 'half' or 'interleaved'")
    dtype = _DTYPES.get(query.dtype)
    if dtype is None:
        raise TypeError('query must be bfloat16 or float32')
    stride = query.stride()
    if len(stride) != 4 or stride[3] != 1:
        raise ValueError('query must be [B, H, N, D] with a contiguous head_dim')
    B, H, N, D = query.shape
    if not 2 <= D <= 256:
        raise ValueError(f'head_dim {D} unsupported (2 to 256)')
    if key is None:
        if key_weight is not None:
            raise ValueError('key_weight needs a key')
    else:
        if key.dtype != query.dtype:
            raise TypeError('query and key must have one type')
        shape = key.shape
        if len(shape) != 4 or key.stride(3) != 1 or shape[0] != B or shape[2] != N or shape[3] != D:
            raise ValueError('key must be [B, Hk, N, D] like query with a contiguous head_dim')
    weight_dtype = None
    for w in (query_weight, key_weight):
        if w is None:
            continue
        code = _DTYPES.get(w.dtype)
        if code is None or weight_dtype not in (None, code):
            raise TypeError('weights must be bfloat16 or float32 alike')
        weight_dtype = code
        if w.shape != (D,) or not w.is_contiguous():
            raise ValueError('weights must be contiguous [head_dim] vectors')
    places = positions.shape
    if positions.dtype not in _WHOLE or (places != (N,) and places != (B, N)):
        raise ValueError(f'positions must be int32 or int64 [N] or [B, N], got {positions.dtype} {tuple(places)}')
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous():
        raise ValueError('frequencies must be a contiguous fp64 vector')
    if not 1 <= frequencies.numel() <= min(D // 2, 128):
        raise ValueError(f'{frequencies.numel()} frequencies do not fit head_dim {D} (at most 128)')
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError('eps must be 0 or more and finite')
    how = positions, frequencies, dtype, weight_dtype or 0, LAYOUTS[layout], float(amplitude), eps
    tracked = False
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:      # (once, not for each tensor)
        tracked = any(t is not None and _tracked(t) for t in (query, key, query_weight, key_weight, *(out or ())))
    if out is None:
        if tracked:
            both = _NormRotary.apply(query, key, query_weight, key_weight, *how)
            return (both, None) if key is None else both
        return _normed(query, key, query_weight, key_weight, (_lib.rows_like(query), _like(key)), *how)
    if tracked:
        raise ValueError('out= takes no part in a gradient')
    if len(out) != 2 or (out[1] is None) != (key is None) or out[0] is None:
        raise ValueError('out must be a pair like the results')
    for x, o in zip((query, key), out):
        if o is None:
            continue
        if o.shape != x.shape or o.dtype != x.dtype or o.stride(-1) != 1 or _lib.stacked(o):
            raise ValueError("out must have its input's shape and type, a contiguous head_dim and a place for every element")
        same = o is x or o.data_ptr() == x.data_ptr() and o.stride() == x.stride()
        if not same and _lib.overlaps(o, x) and not _lib.apart(o, x):
            raise ValueError('out must be its input itself or memory that neither input shares')
        if _lib.overlaps_any(o, query_weight, key_weight, positions, frequencies):
            raise ValueError('out must not share memory with weights, positions or frequencies')
    # A side's result and the other side, whose rows other workgroups read and write, be it the same tensor.
    first, second = out
    crossed = [(first, key)]
    if second is not key:
        crossed.append((first, second))
    if first is not query or second is not key:
        crossed.append((second, query))
    for a, b in crossed:
        if b is not None and a is not None and _lib.overlaps(a, b) and not _lib.apart(a, b):
            raise ValueError('out must not share memory with the other input or the other result')
    return _normed(query, key, query_weight, key_weight, tuple(out), *how)

