"""Rotary positions of one axis on the HIP kernels: interleaved and half layouts, part of a head, frequencies scaled for
contexts longer than the trained one.

Beside `producer.axial_rope` (AxialRoPE, streamvoxel/models/unconditional_md4.py:10-24), which turns the three axes of
the reference's positions with the reference's bf16 roundings; no counterpart in the reference.
"""
from __future__ import annotations

import math
import struct

import torch
from torch.autograd import forward_ad

from streamvoxel_amd import _lib

__all__ = ['rotary', 'rotary_frequencies']

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
    return _launch(x, torch.empty_like(x), positions, frequencies, layout, amplitude, inverse)


class _Rotary(torch.autograd.Function):
    """The rotation, or its transpose (inverse 1): linear, so that each is the other's gradient, as often as asked for,
    and a tangent turns as x does."""

    @staticmethod
    def forward(ctx, x, positions, frequencies, layout, amplitude, inverse):
        ctx.save_for_backward(positions, frequencies)
        ctx.save_for_forward(positions, frequencies)
        ctx.args = layout, amplitude, inverse
        return _launch(x, torch.empty_like(x), positions, frequencies, layout, amplitude, inverse)

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
        out = torch.empty_like(x)
    else:
        if _tracked(x) or _tracked(out):
            raise ValueError('out= takes no part in a gradient')
        if out.shape != x.shape or out.dtype != x.dtype or out.stride(-1) != 1 or _lib.stacked(out):
            raise ValueError("out must have x's shape and type, a contiguous head_dim and a place for every element")
        if _lib.overlaps(x, out) and (x.data_ptr() != out.data_ptr() or x.stride() != out.stride()):
            raise ValueError('out must be x itself or memory that x does not share')
    return _launch(x, out, positions, frequencies, layout, float(amplitude), 0)
