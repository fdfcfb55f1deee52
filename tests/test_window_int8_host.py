"""CPU checks of the int8 paged cache, the reading back, the window and the normed rotation: the refusals of the C ABI (no
launch) and of the Python entry points."""
import math
import os
import struct

import pytest
import torch

from streamvoxel_amd import _lib
from streamvoxel_amd.stream.paged import PagedContext, paged_attention, paged_read
from streamvoxel_amd.stream.rotary import norm_rotary

FAKE = 0x1000      # never dereferenced: every call below fails its host checks, or launches nothing


@pytest.fixture(scope='module')
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from streamvoxel_amd.build import build
        build()
    return _lib.load()


def cache_of(dtype=17, B=2, H=2, D=64, ke=FAKE, ve=FAKE, pages=4, page=64, kp=FAKE, lengths=FAKE, table=FAKE, srow=64, m=2):
    return struct.pack('7P18q', kp, FAKE, ke, ve, table, lengths, 0, dtype, B, H, D, pages, page, m, m, 8192, 4096, srow, 8192, 4096,
                       srow, 4, 2, 4, 2)


def read_args(key=FAKE, value=FAKE, N=3, before=0, strides=(1024, 512, 64)):
    return struct.pack('3P8q', key, value, 0, N, before, *strides, *strides)


def attend_args(q=FAKE, out=FAKE, ws=FAKE, nbytes=1 << 40, H=4, N=1, causal=1, scale=1.0, stride=64):
    return struct.pack('4P10qd', q, out, 0, ws, nbytes, H, N, *[stride] * 6, causal, scale)


def append_args(N=1):
    return struct.pack('5P13qd', FAKE, FAKE, 0, 0, 0, N, 0, *[64] * 6, 0, 0, 0, 0, 0, 1.0)


def test_int8_caches(lib):
    calls = (lambda c: lib.svhip_paged_read(c, read_args(), None), lambda c: lib.svhip_paged_append(c, append_args(), None),
             lambda c: lib.svhip_paged_attention(c, attend_args(), None),
             lambda c: lib.svhip_paged_window_attention(c, attend_args(), 5, 1, None))
    for call in calls:
        for dtype in (0, 2, 5, 15, 19):
            assert call(cache_of(dtype)) == -1 and b'dtype' in lib.svhip_last_error()
        for dtype, page in ((17, 16), (18, 16), (18, 32)):
            assert call(cache_of(dtype, page=page)) == -1 and b'block' in lib.svhip_last_error()
        for dtype in (16, 17, 18, 3):
            assert call(cache_of(dtype, ke=0)) == -1 and b'exponents' in lib.svhip_last_error()
            assert call(cache_of(dtype, ve=0)) == -1 and b'exponents' in lib.svhip_last_error()
            assert call(cache_of(dtype, kp=FAKE + 4)) == -1 and b'boundaries' in lib.svhip_last_error()
        for c in (cache_of(B=0), ):
            assert call(c) == 0
        assert call(None) == -1 and b'null' in lib.svhip_last_error()


def test_read_refusals(lib):
    read = lambda args, c=cache_of(): lib.svhip_paged_read(c, args, None)
    assert read(read_args(key=0)) == -1 and b'null' in lib.svhip_last_error()
    assert read(read_args(value=0)) == -1 and b'null' in lib.svhip_last_error()
    assert read(None) == -1 and b'null' in lib.svhip_last_error()
    for how in (dict(N=-1), dict(before=-1), dict(N=1 << 31), dict(before=1 << 31)):
        assert read(read_args(**how)) == -1 and b'sizes' in lib.svhip_last_error()
    for how in (dict(key=FAKE + 8), dict(value=FAKE + 2), dict(strides=(1024, 512, 68)), dict(strides=(1024, 516, 64))):
        assert read(read_args(**how)) == -1 and b'16-byte' in lib.svhip_last_error()
    assert read(read_args(N=0)) == 0
    assert read(read_args(N=(1 << 30) + 1), cache_of(B=2)) == -1 and b'large' in lib.svhip_last_error()
    assert read(read_args(), cache_of(lengths=0)) == -1 and b'null' in lib.svhip_last_error()
    assert read(read_args(), cache_of(pages=0)) == -1 and b'page' in lib.svhip_last_error()


def test_window_refusals(lib):
    call = lambda window, sinks, dtype=1, **how: lib.svhip_paged_window_attention(
        cache_of(dtype, kp=0x2000), attend_args(**how), window, sinks, None)
    for window, sinks in ((0, 0), (-1, 0), (5, -1)):
        assert call(window, sinks) == -1 and b'window' in lib.svhip_last_error()
    assert call(5, 0, causal=0) == -1 and b'causal' in lib.svhip_last_error()
    assert call(5, 0, N=0) == 0 and call(1 << 62, 1 << 62, N=0) == 0
    assert call(5, 0, q=0) == -1 and b'null' in lib.svhip_last_error()
    assert call(5, 0, scale=math.nan) == -1 and b'scale' in lib.svhip_last_error()
    need = lib.svhip_paged_attention_workspace_bytes(2, 4, 2, 200, 0, 64, 64 * 64)
    for ws, nbytes in ((0, need), (FAKE, 64), (FAKE + 8, need)):
        args = attend_args(ws=ws, nbytes=nbytes, N=200)
        assert lib.svhip_paged_window_attention(cache_of(1, m=64), args, 3000, 0, None) == -1
        assert b'workspace' in lib.svhip_last_error()
    assert lib.svhip_paged_window_attention(cache_of(), None, 5, 0, None) == -1 and b'null' in lib.svhip_last_error()


def norm_args(q=FAKE, k=FAKE, dq=FAKE, dk=FAKE, out=FAKE, dwq=0, dwk=0, positions=FAKE, freq=FAKE, ws=0, nbytes=0, dtype=1, wdtype=1,
              pairs=32, layout=1, sizes=(1, 4, 2, 3, 64), amplitude=1.0, eps=1e-6):
    return struct.pack('13P31q2d', q, k, dq, dk, FAKE, FAKE, out, out, dwq, dwk, positions, freq, ws, nbytes, dtype, wdtype, 0, pairs,
                       layout, *sizes, *[64] * 18, 0, 1, amplitude, eps)


@pytest.mark.parametrize('name', ['svhip_norm_rotary', 'svhip_norm_rotary_grad'])
def test_norm_rotary_refusals(lib, name):
    call = lambda **how: getattr(lib, name)(norm_args(**how), None)
    grad = name.endswith('grad')
    for how in (dict(q=0), dict(k=0), dict(positions=0), dict(freq=0), dict(dq=0) if grad else dict(out=0)):
        assert call(**how) == -1 and b'null' in lib.svhip_last_error(), how
    for how in (dict(dtype=3), dict(wdtype=3), dict(dtype=16)):
        assert call(**how) == -1 and b'dtype' in lib.svhip_last_error()
    for how in (dict(layout=0), dict(layout=3)):
        assert call(**how) == -1 and b'layout' in lib.svhip_last_error()
    for how in (dict(pairs=0), dict(pairs=33), dict(pairs=129, sizes=(1, 1, 1, 1, 256))):
        assert call(**how) == -1 and b'pairs' in lib.svhip_last_error()
    for D in (1, 257, 0, 1 << 20):
        assert call(sizes=(1, 1, 1, 1, D)) == -1 and b'head_dim' in lib.svhip_last_error()
    for sizes in ((-1, 1, 1, 1, 64), (1, -1, 1, 1, 64), (1, 1, -1, 1, 64), (1, 1, 1, -1, 64), (1 << 31, 1, 1, 1, 64)):
        assert call(sizes=sizes) == -1 and b'sizes' in lib.svhip_last_error()
    for eps in (-1.0, math.nan, math.inf):
        assert call(eps=eps) == -1 and b'eps' in lib.svhip_last_error()
    for sizes in ((0, 1, 1, 1, 64), (1, 0, 0, 1, 64), (1, 1, 1, 0, 64)):
        assert call(sizes=sizes) == 0
    if grad:
        need = lib.svhip_norm_rotary_workspace_bytes(1, 4, 2, 3, 64)
        assert need >= 2 * 3 * 64 * 4
        for how in (dict(ws=0, nbytes=need), dict(ws=FAKE, nbytes=64 * 4), dict(ws=FAKE + 2, nbytes=need)):
            assert call(dwq=FAKE, **how) == -1 and b'workspace' in lib.svhip_last_error()
    assert getattr(lib, name)(None, None) == -1 and b'null' in lib.svhip_last_error()
    assert lib.svhip_norm_rotary_workspace_bytes(0, 1, 1, 3, 64) == lib.svhip_norm_rotary_workspace_bytes(1, 0, 0, 3, 64) == 0
    assert lib.svhip_norm_rotary_workspace_bytes(1 << 20, 8, 8, 1 << 20, 256) == 768 * 2 * 256 * 4


def test_host_tensors_are_refused():
    x, w = torch.zeros(1, 2, 3, 8, dtype=torch.bfloat16), torch.ones(8)
    pages, table, n = torch.zeros(2, 2, 16, 8, dtype=torch.int8), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    e = torch.ones(2, 2, 1, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match='GPU'):
        norm_rotary(x, x, w, w, torch.zeros(3, dtype=torch.int32), torch.ones(4, dtype=torch.float64))
    with pytest.raises(RuntimeError, match='GPU'):
        paged_read(pages, pages, table, n, 3, k_exponents=e, v_exponents=e)
    with pytest.raises(RuntimeError, match='GPU'):
        paged_attention(x, pages, pages, table, n, causal=True, window=5, k_exponents=e, v_exponents=e)


@pytest.mark.parametrize('args', [dict(kv_dtype='int4'), dict(kv_dtype='int8', block=8), dict(kv_dtype='int8', block=128, page_size=128),
                                  dict(kv_dtype='int8', block=64, page_size=32), dict(kv_dtype='bf16', block=16)])
def test_paged_context_refusals(args):
    with pytest.raises(ValueError):
        PagedContext(1, 1, 1, 64, 4, 'cpu', **args)


@pytest.mark.parametrize('page, block, rows', [(64, None, 1), (16, None, 1), (128, None, 2), (64, 16, 4), (32, 32, 1)])
def test_paged_context_has_an_exponent_a_block(page, block, rows):
    ctx = PagedContext(2, 1, 3, 64, 4, 'cpu', page_size=page, kv_dtype='int8', block=block)
    assert ctx.k[0].dtype == torch.int8 and ctx.k_exponents[1].shape == ctx.v_exponents[0].shape == (4, 3, rows)


def test_int8_needs_pages():
    from streamvoxel_amd.stream.engine import check_engine_options
    check_engine_options('gather', 'flex', False, 'int8', paged=True)
    with pytest.raises(ValueError, match='pages'):
        check_engine_options('gather', 'flex', False, 'int8')


def test_tensors_that_lie_apart():
    base = torch.zeros(2, 5, 12, 64)
    q, k, v = [base[:, :, i:j].transpose(1, 2) for i, j in ((0, 8), (8, 10), (10, 12))]
    assert _lib.apart(q, k) and _lib.apart(k, q) and _lib.apart(q, v) and _lib.apart(k, v)
    assert not _lib.apart(q, q) and not _lib.apart(q, base[:, :, 7:9].transpose(1, 2)) and not _lib.apart(q, q[:, 1:3])
    first, second = torch.zeros(2, 6, 5, 8).chunk(2, 1)
    assert _lib.apart(first, second) and not _lib.apart(first, second.transpose(1, 2))
    pair = torch.zeros(7, 2, 3, 8)
    assert _lib.apart(pair[:, 0], pair[:, 1]) and _lib.apart(pair[:, 0].transpose(0, 1), pair[:, 1].transpose(0, 1))
    one = torch.zeros(1, 1, 12, 64)
    assert _lib.apart(one[:, :, :8].transpose(1, 2), one[:, :, 8:].transpose(1, 2))
    flat = torch.zeros(100)
    a, b = flat.as_strided((3, 4), (10, 2)), flat.as_strided((3, 4), (10, 2), 1)
    assert _lib.apart(a, b)                                     # every other element of each
    assert not _lib.apart(flat.as_strided((3, 6), (10, 2)), flat.as_strided((3, 6), (10, 2), 1))     # a row's end past the next's start
    assert not _lib.apart(flat.as_strided((3,), (0,)), flat.as_strided((3,), (0,), 1))
    g = torch.Generator().manual_seed(1)                         # against the elements themselves
    draw = lambda low, high: int(torch.randint(low, high, (1,), generator=g))
    seen = [0, 0]
    for _ in range(3000):
        stride = (draw(1, 14), draw(1, 6))
        shapes = [(draw(1, 4), draw(1, 5)) for _ in 'ab']
        a, b = [flat.as_strided(shape, stride, at) for shape, at in zip(shapes, (0, draw(0, 12)))]
        places = [set((t.storage_offset() + i * t.stride(0) + j * t.stride(1)) for i in range(t.shape[0]) for j in range(t.shape[1]))
                  for t in (a, b)]
        if _lib.apart(a, b):
            seen[0] += 1
            assert not places[0] & places[1]
        else:
            seen[1] += 1
    assert min(seen) > 200


@pytest.mark.parametrize('stride', [(24, 8, 1, 1), (1, 1, 1, 1), (100, 1, 8, 1), (64, 16, 8, 1), (0, 0, 0, 1), (96, 8, 24, 1)], ids=str)
def test_results_of_rows_that_overlap_have_a_contiguous_head_dim(stride):
    x = torch.empty(400).as_strided((2, 3, 4, 8), stride)
    y = _lib.rows_like(x)
    assert y.shape == x.shape and y.stride(-1) == 1 and not _lib.stacked(y)
    assert len({sum(i * s for i, s in zip(at, y.stride())) for at in torch.cartesian_prod(*map(torch.arange, x.shape)).tolist()}) == 192
