"""The int8 append on the GPU from 1024 tokens on, where a workgroup has several tokens and several blocks begin among them, and
with positions and an amplitude of its own; against plain float64 on the host.

Tolerances: those of test_gpu_paged_int8.py, and for far positions that of the phase p f itself. The kernel forms its turns
p (f / 2 pi) in 64 bits, three roundings of 2^-53 (the constant's, two products'), the reference p f with one: together
4 * 2^-53 |p| f radians, which move an element by that much of its pair's |a| + |b| (2^-11 of it at position 2^40, nothing
beside 8 * 2^-24 below 2^25)."""
import math

import pytest
import torch

import test_gpu_paged_int8 as base

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
E = 2.0 ** -24


@pytest.mark.parametrize('layout, part', [(None, 0), ('half', 1.0), ('interleaved', 0.3)])
@pytest.mark.parametrize('D, H, page, block', [(8, 1, 32, 16), (48, 2, 16, 16), (64, 1, 64, 32)])
@pytest.mark.parametrize('counts, packed, before', [([1] * 1100, False, 0), ([3] * 700, False, 2), ([600, 1, 0, 800, 33, 1], True, 0),
                                                    ([1] * 900 + [90] + [2] * 300, True, 0)], ids=['ones', 'threes', 'long', 'mixed'])
def test_slots_of_several_tokens(counts, packed, before, D, H, page, block, layout, part):
    base.test_append_against_float64(counts, packed, before, D, H, page, block, layout, part)


@pytest.mark.parametrize('layout', [None, 'half', 'interleaved'])
@pytest.mark.parametrize('total', [17000, 33001])
def test_slots_that_several_blocks_begin_in(total, layout):
    """Up to 64 tokens a workgroup: four blocks of 16 of one window."""
    base.test_append_against_float64([total - 700, 3, 697], True, 0, 8, 2, 64, 16, layout, 1.0)


@pytest.mark.parametrize('amplitude', [1.0, -1.3, 0.25])
@pytest.mark.parametrize('wide', [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize('packed', [False, True])
@pytest.mark.parametrize('layout, half', [('half', 32), ('half', 11), ('interleaved', 32), ('interleaved', 20)])
@pytest.mark.parametrize('n', [1, 100, 1300])
def test_positions_and_amplitudes(n, layout, half, packed, wide, amplitude):
    """Positions anywhere (strided, beyond 2^31 where they are wide) and a scaled rotation: what is held lies within half a step of
    the turned key, and the block's power of two is the least that holds it."""
    from streamvoxel_amd.stream.paged import paged_append, paged_read
    base._case(f'int8 append positions n={n} {layout} {half} packed={packed} {wide} {amplitude}')
    B, H, D, page, block = 2, 2, 64, 64, 32
    g = torch.Generator().manual_seed(n + half)
    key, value = [torch.randn(B, H, n, D, generator=g).to(torch.bfloat16) for _ in 'kv']
    far = 1 << 40 if wide == torch.int64 else 1 << 20
    where = torch.randint(-far, far, (B, n, 2), generator=g).to(wide)[..., 1]           # (every other element)
    freq = 100.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    pages = -(-n // page)
    table = torch.randperm(B * pages, generator=g).to(torch.int32).view(B, pages).to(DEV)
    k, v = [torch.zeros(B * pages, H, page, D, dtype=torch.int8, device=DEV) for _ in 'kv']
    e = {name: torch.zeros(B * pages, H, page // block, dtype=torch.uint8, device=DEV) for name in ('k_exponents', 'v_exponents')}
    L = torch.full((B,), n, dtype=torch.int32, device=DEV)
    rows = lambda t: (t.transpose(0, 1).reshape(H, B * n, D) if packed else t).to(DEV)
    spaced = torch.stack([where, where], -1).to(DEV)[..., 0]
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=DEV) if packed else None
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    paged_append(rows(key), rows(value), k, v, table, L, cu_tokens=cu, bad=bad, frequencies=freq.to(DEV), layout=layout,
                 amplitude=amplitude, positions=spaced.flatten() if packed else spaced, **e)
    assert int(bad) == 0
    got = paged_read(k, v, table, L, n, **e)
    scale = torch.ones(D, dtype=torch.float64)
    scale[:2 * half] = amplitude
    for b in range(B):
        x = key[b].double()
        turned, off = base.turned64(x, where[b], freq, layout)
        far_off = 4 * 2.0 ** -53 * where[b].double().abs()[:, None] * freq                # (off is 8 E (|a| + |b|))
        for at in (slice(0, half), slice(half, 2 * half)) if layout == 'half' else (slice(0, 2 * half, 2), slice(1, 2 * half, 2)):
            off[..., at] = off[..., at] * (1 + far_off / (8 * E))
        turned, off = turned * scale, off * scale.abs()
        at = table[b].cpu().long()
        exponent = e['k_exponents'].cpu()[at].transpose(0, 1).reshape(H, -1)[:, :-(-n // block)]
        power = 2.0 ** (exponent.double() - 127)
        step = power.repeat_interleave(block, -1)[:, :n, None]
        assert ((got[0][b].cpu().double() - turned).abs() <= step / 2 + off).all(), b
        most = torch.nn.functional.pad((turned.abs() + off).amax(-1), (0, -n % block)).unflatten(-1, (-1, block)).amax(-1)
        assert (most * (1 + 16 * E) > 127 * power / 2).all() and ((turned.abs() - off) <= 127 * step).all()
        steps = 2.0 ** (e['v_exponents'].cpu()[at].transpose(0, 1).reshape(H, -1)[:, :-(-n // block)].double() - 127)
        assert ((got[1][b].cpu().double() - value[b].double()).abs() <= steps.repeat_interleave(block, -1)[:, :n, None] / 2).all()
