"""CPU checks of the rotary positions and the paged cache: the frequencies, the refusals of the C ABI (no launch) and of the
Python entry points."""
import struct
import math

import pytest
import torch

from streamvoxel_amd import _lib
from streamvoxel_amd.stream.rotary import rotary, rotary_frequencies


@pytest.fixture(scope='module')
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from streamvoxel_amd.build import build
        build()
    return _lib.load()


def test_rotary_frequencies():
    f, a = rotary_frequencies(8, base=100.0)
    assert a == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-14, atol=0)
    assert torch.equal(rotary_frequencies(8, base=100.0, scaling='linear', factor=4.0)[0], f / 4)
    g, a = rotary_frequencies(64, scaling='wavelength', factor=8.0, original_length=2048)
    f = rotary_frequencies(64)[0]
    assert abs(a - (0.1 * math.log(8) + 1)) < 1e-15
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(g[turns > 32], f[turns > 32])
    assert torch.allclose(g[turns < 1], f[turns < 1] / 8, rtol=1e-14, atol=0)
    assert (g[1:] < g[:-1]).all() and (g <= f).all() and (g >= f / 8 * (1 - 1e-14)).all()
    assert torch.equal(rotary_frequencies(64, scaling='wavelength', original_length=2048)[0], f)     # factor 1


@pytest.mark.parametrize('args', [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling='cubic'),
                                  dict(rotary_dim=8, scaling='linear', factor=0.5),
                                  dict(rotary_dim=8, scaling='wavelength', factor=2.0),
                                  dict(rotary_dim=8, scaling='wavelength', original_length=100, low=4.0, high=4.0)])
def test_rotary_frequencies_refusals(args):
    with pytest.raises(ValueError):
        rotary_frequencies(**args)


def test_host_tensors_are_refused():
    from streamvoxel_amd.stream.paged import paged_append, paged_attention
    x = torch.zeros(1, 2, 3, 8, dtype=torch.bfloat16)
    pages, table, n = torch.zeros(2, 2, 16, 8, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32), torch.ones(
        1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match='GPU'):
        rotary(x, torch.zeros(3, dtype=torch.int32), torch.ones(4, dtype=torch.float64))
    with pytest.raises(RuntimeError, match='GPU'):
        paged_append(x, x, pages, pages, table, n)
    with pytest.raises(RuntimeError, match='GPU'):
        paged_attention(x, pages, pages, table, n)


FAKE = 0x1000      # never dereferenced: every call below fails its host checks, or launches nothing


def test_rotary_argument_errors(lib):
    def call(x=FAKE, dtype=1, freq=FAKE, pairs=4, layout=1, sizes=(1, 2, 3, 8)):
        args = struct.pack('4P17qd', x, FAKE, FAKE, freq, dtype, 0, pairs, layout, 0, *sizes, *[8] * 6, 0, 1, 1.0)
        return lib.svhip_rotary(args, None)
    assert call(x=0) == -1 and b'null' in lib.svhip_last_error()
    assert call(freq=0) == -1 and b'null' in lib.svhip_last_error()
    assert call(dtype=3) == -1 and b'dtype' in lib.svhip_last_error()
    for layout in (0, 3, 9):
        assert call(layout=layout) == -1 and b'layout' in lib.svhip_last_error()
    for pairs, D in ((5, 8), (0, 8), (129, 512)):
        assert call(pairs=pairs, sizes=(1, 2, 3, D)) == -1 and b'pairs' in lib.svhip_last_error()
    assert call(sizes=(1, 2, -3, 8)) == -1 and b'sizes' in lib.svhip_last_error()
    for sizes in ((0, 2, 3, 8), (1, 0, 3, 8), (1, 2, 0, 8)):
        assert call(sizes=sizes) == 0
    assert lib.svhip_rotary(None, None) == -1 and b'null' in lib.svhip_last_error()


def cache_of(B=2, H=2, D=64, kp=FAKE, ke=0, dtype=1, pages=4, page=64, srow=64, table=FAKE, m=2, lengths=FAKE):
    return struct.pack('7P18q', kp, FAKE, ke, ke, table, lengths, 0, dtype, B, H, D, pages, page, m, m, 8192, 4096, srow,
                       8192, 4096, srow, 128, 64, 128, 64)


def append_call(lib, key=FAKE, sk=(768, 64, 128), N=3, before=0, layout=0, positions=0, freq=0, pairs=0, **cache):
    args = struct.pack('5P13qd', key, FAKE, 0, positions, freq, N, before, *sk, 768, 64, 128, layout, 0, 6, 1, pairs, 1.0)
    return lib.svhip_paged_append(cache_of(**cache), args, None)


def attend_call(lib, q=FAKE, H=4, N=3, sq=64, so=64, scale=0.125, ws=0, nbytes=0, **cache):
    args = struct.pack('4P10qd', q, FAKE, 0, ws, nbytes, H, N, 768, 192, sq, 768, 192, so, 0, scale)
    return lib.svhip_paged_attention(cache_of(**cache), args, None)


@pytest.mark.parametrize('call', [append_call, attend_call])
def test_cache_errors(lib, call):
    error = lib.svhip_last_error
    for D in (0, 60, 136):
        assert call(lib, D=D) == -1 and b'head_dim' in error()
    for page in (0, 8, 48, 2048):
        assert call(lib, page=page) == -1 and b'page size' in error()
    assert call(lib, dtype=0) == -1 and b'dtype' in error()
    assert call(lib, B=-1) == -1 and b'sizes' in error()
    for kw in (dict(pages=-1), dict(m=-1), dict(m=1 << 25), dict(pages=1 << 31)):
        assert call(lib, **kw) == -1 and b'page counts' in error()
    assert call(lib, pages=0) == -1 and b'needs a page' in error()
    for name in ('kp', 'table', 'lengths'):
        assert call(lib, **{name: 0}) == -1 and b'null' in error()
    assert call(lib, dtype=3) == -1 and b'exponents' in error()
    assert call(lib, srow=68) == -1 and b'16-byte' in error()
    assert call(lib, dtype=3, ke=FAKE, srow=68) == -1 and b'8-byte' in error()
    for srow in (-64, 1 << 24):
        assert call(lib, srow=srow) == -1 and b'too far' in error()
    for empty in (dict(B=0), dict(N=0)):
        assert call(lib, **empty) == 0


def test_append_argument_errors(lib):
    error = lib.svhip_last_error
    assert append_call(lib, before=-1) == -1 and b'sizes' in error()
    assert append_call(lib, layout=4) == -1 and b'layout' in error()
    assert append_call(lib, layout=1, freq=FAKE, pairs=33) == -1 and b'pairs' in error()
    assert append_call(lib, layout=2, freq=FAKE, pairs=0) == -1 and b'pairs' in error()
    assert append_call(lib, layout=1, pairs=32) == -1 and b'frequencies' in error()
    assert append_call(lib, layout=3, freq=FAKE, positions=FAKE, pairs=32) == -1 and b'three-axis' in error()
    assert append_call(lib, layout=3, freq=FAKE, pairs=24, D=48) == -1 and b'positions' in error()
    assert append_call(lib, key=0) == -1 and b'null' in error()
    assert append_call(lib, sk=(768, 60, 128)) == -1 and b'16-byte' in error()
    assert append_call(lib, H=0) == 0
    assert lib.svhip_paged_append(None, None, None) == -1 and b'null' in error()
    assert lib.svhip_paged_append(cache_of(), None, None) == -1 and b'null' in error()


def test_attention_argument_errors(lib):
    error = lib.svhip_last_error
    for heads in (0, 3):
        assert _attend_heads(lib, heads) == -1 and b'share' in error()
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert attend_call(lib, scale=scale) == -1 and b'scale' in error()
    assert attend_call(lib, N=-1) == -1 and b'sizes' in error()
    assert attend_call(lib, q=0) == -1 and b'null' in error()
    assert attend_call(lib, sq=68) == -1 and b'query rows' in error()
    assert attend_call(lib, so=66) == -1 and b'rows of out' in error()
    assert lib.svhip_paged_attention_workspace_bytes(2, 4, 2, 3, 0, 64, 128) == 0     # too few keys for parts
    need = lib.svhip_paged_attention_workspace_bytes(2, 4, 2, 3, 0, 64, 1280)
    assert need > 0
    for ws, nbytes in ((0, need), (FAKE, need - 1), (FAKE + 8, need)):
        assert attend_call(lib, m=20, ws=ws, nbytes=nbytes) == -1 and b'workspace' in error()
    assert lib.svhip_paged_attention(None, None, None) == -1 and b'null' in error()
    assert lib.svhip_paged_attention(cache_of(), None, None) == -1 and b'null' in error()


def _attend_heads(lib, heads):
    args = struct.pack('4P10qd', FAKE, FAKE, 0, 0, 0, 4, 3, 768, 192, 64, 768, 192, 64, 0, 0.125)
    return lib.svhip_paged_attention(cache_of(H=heads), args, None)


def test_workspace_query():
    """Bytes for what a call may launch; nothing for sizes that no call takes."""
    need = _lib.load().svhip_paged_attention_workspace_bytes
    assert need(0, 4, 2, 3, 0, 64, 128) == need(2, 4, 3, 3, 0, 64, 128) == need(2, 4, 2, 0, 0, 64, 128) == 0
    assert need(8, 12, 12, 1024, 0, 64, 9744) == 0           # tiles that fill the chip
    assert need(1, 12, 12, 1024, 0, 64, 9744) > 0
    assert need(64, 16, 16, 1, 0, 64, 9744) > 0


def test_paged_context_books(monkeypatch):
    """The pages that windows take, keep and give back, without a device."""
    from streamvoxel_amd.stream.paged import PagedContext
    monkeypatch.setattr(PagedContext, '_send', staticmethod(lambda to, v: to.copy_(torch.tensor(v, dtype=torch.int32))))
    ctx = PagedContext(2, 3, 2, 64, 8, 'cpu', page_size=16, max_pages=5)
    assert len(ctx.k) == len(ctx.v) == 2 and ctx.k[0].shape == (8, 2, 16, 64) and ctx.k_exponents == [None, None]
    ctx.resize(0, 33)
    ctx.resize(1, 16)
    assert ctx.table[0, :3].tolist() == ctx._owned[0] == [0, 1, 2] and ctx._owned[1] == [3] and ctx.free_pages == 4
    ctx.grow((15, 0, 1))
    assert ctx.lengths.tolist() == ctx.host_lengths == [48, 16, 1] and ctx._owned[0] == [0, 1, 2] and ctx._owned[2] == [4]
    ctx.grow(1)
    assert ctx._owned[0] == [0, 1, 2, 5] and ctx._owned[1] == [3, 6] and ctx.free_pages == 1
    ctx.resize(0, 20)
    assert ctx._owned[0] == [0, 1] and ctx.free_pages == 3 and ctx.lengths.tolist() == [20, 17, 2]
    ctx._set({1: 0, 2: 80})                      # pages given back in the same call serve the other window
    assert ctx.free_pages == 1 and len(ctx._owned[2]) == 5 and ctx._owned[1] == []
    assert sorted(sum(ctx._owned, ctx._free[:])) == list(range(8))
    assert ctx.table[2].tolist() == ctx._owned[2]
    e = PagedContext(1, 1, 2, 64, 3, 'cpu', kv_dtype='fp8')
    assert e.max_pages == 3 and e.k[0].dtype == torch.float8_e4m3fn and e.k_exponents[0].shape == (3, 2, 64)


@pytest.mark.parametrize('args', [dict(kv_dtype='fp16'), dict(page_size=24), dict(page_size=8), dict(head_dim=60),
                                  dict(head_dim=136), dict(pages=0), dict(max_pages=0), dict(batch=0)])
def test_paged_context_refusals(args):
    from streamvoxel_amd.stream.paged import PagedContext
    with pytest.raises(ValueError):
        PagedContext(**{**dict(layers=1, batch=1, heads=2, head_dim=64, pages=4, device='cpu'), **args})


def test_pages_of_an_engine_need_its_paged_context():
    from streamvoxel_amd.stream.engine import SlotEngine, check_engine_options
    assert check_engine_options('gather', 'flex', False) is None
    with pytest.raises(RuntimeError, match='HIP'):
        SlotEngine(None, None, 'cpu', 1, 1, 1, pages=4)


def test_sizes_that_would_not_fit_the_kernels_counts(lib):
    """Key numbers, a few blocks past the last of them, stay below 2^31; windows, tokens and heads are bounded."""
    error = lib.svhip_last_error
    for call in (append_call, attend_call):
        for m, page in (((1 << 24) + 1, 64), ((1 << 20) + 1, 1024)):
            assert call(lib, m=m, page=page) == -1 and b'page counts' in error()
        for kw in (dict(B=1 << 31), dict(H=(1 << 20) + 1), dict(N=1 << 31)):
            assert call(lib, **kw) == -1 and b'sizes' in error()
    assert append_call(lib, before=1 << 31) == -1 and b'sizes' in error()
    for sizes in ((1 << 31, 1, 1, 8), (1, 1, 1 << 31, 8)):
        args = struct.pack('4P17qd', FAKE, FAKE, FAKE, FAKE, 1, 0, 4, 1, 0, *sizes, *[8] * 6, 0, 1, 1.0)
        assert lib.svhip_rotary(args, None) == -1 and b'sizes' in error()
    need = lib.svhip_paged_attention_workspace_bytes
    assert need(2, 4, 2, 3, 0, 64, (1 << 30) + 1) == need(1 << 31, 4, 2, 3, 0, 64, 1280) == 0
    assert need(2, 1 << 20, 2, 1 << 21, 0, 64, 1280) == 0


class Streams:
    """Stands in for the device of a PagedContext on the CPU: what is sent on stream `late` happens at `catch_up` alone, what
    is sent on stream `now` at once."""

    def __init__(self, monkeypatch):
        from streamvoxel_amd.stream.paged import PagedContext
        self.current, self.queue = 'now', []
        monkeypatch.setattr(PagedContext, '_send', staticmethod(self.send))

    def send(self, to, values):
        values = torch.tensor(values, dtype=torch.int32)
        if self.current == 'late':
            self.queue.append(lambda: to.copy_(values))
        else:
            to.copy_(values)

    def catch_up(self):
        for work in self.queue:
            work()
        self.queue.clear()


def test_a_window_in_work_on_another_stream_leaves_the_other_lengths_alone(monkeypatch):
    from streamvoxel_amd.stream.paged import PagedContext
    streams = Streams(monkeypatch)
    ctx = PagedContext(1, 8, 2, 64, 40, 'cpu', page_size=16)
    ctx.grow(10)
    for change in (lambda: ctx.resize(1, 20), lambda: ctx.grow((0, 30, 0, 0, 0, 0, 0, 0)), lambda: ctx.release(1)):
        streams.current = 'late'
        change()
        streams.current = 'now'
        ctx.grow((1, 0, 1, 1, 0, 1, 0, 1))
        ctx.resize(4, ctx.host_lengths[4] + 3)
        ctx.release(6)
        streams.catch_up()
        assert ctx.lengths.tolist() == ctx.host_lengths
        for b in range(8):
            assert ctx.table[b, :len(ctx._owned[b])].tolist() == ctx._owned[b]


class RecordedStream:
    """A stream that keeps a list of what is put on it."""

    def __init__(self, name):
        self.name, self.work = name, []

    def record_event(self):
        self.work.append('event')
        return self.name, len(self.work)

    def wait_event(self, event):
        self.work.append(('wait', event))


def test_a_page_that_changes_streams_is_waited_for(monkeypatch):
    """The stream that takes a page waits for the one that gave it back, before it sends the table; pages that stay on a
    stream, or were never given back, cost no wait."""
    from streamvoxel_amd.stream.paged import PagedContext
    side, main = RecordedStream('side'), RecordedStream('main')
    current = [side]
    monkeypatch.setattr(PagedContext, '_stream', lambda self: current[0])

    def send(to, values):
        if values:
            current[0].work.append('send')
            to.copy_(torch.tensor(values, dtype=torch.int32))
    monkeypatch.setattr(PagedContext, '_send', staticmethod(send))
    ctx = PagedContext(1, 3, 2, 64, 6, 'cpu', page_size=16)
    ctx.resize(0, 64)
    assert side.work == ['send', 'send']
    side.work.append('keys of window 0')
    ctx.resize(0, 10)                        # three pages back
    assert side.work[2:] == ['keys of window 0', 'event', 'send', 'send']
    current[0] = main
    ctx.resize(1, 33)
    assert ctx._owned[1] == [1, 2, 3] and main.work == [('wait', ('side', 4)), 'send', 'send']
    main.work.clear()
    ctx.resize(2, 30)                        # never used before
    assert main.work == ['send', 'send']
    main.work.clear()
    ctx.release(1)
    ctx.resize(2, 60)                        # given back on this stream
    assert main.work == ['event', 'send', 'send', 'send']
    current[0] = side
    side.work.clear()
    ctx.resize(0, 17)
    assert side.work == [('wait', ('main', 1)), 'send', 'send'] and not ctx._left


class Layer(torch.nn.Module):
    def __init__(self, width, context_width, heads):
        super().__init__()
        self.heads, self.width = heads, width
        self.key_value = torch.nn.Linear(context_width, 2 * width)
        self.rope = torch.nn.Module()
        self.rope.frequencies = torch.ones(width // heads // 6)


@pytest.mark.filterwarnings('ignore:.*autocast')
@pytest.mark.parametrize('fails', [None, 'width', 'layer'])
def test_a_slot_is_extended_whole_or_not_at_all(fails, monkeypatch):
    """The new keys are written under a length of their own; the slot's stays what it was until the last layer has them, and
    for good, its pages too, when one fails."""
    from streamvoxel_amd.stream import paged
    from streamvoxel_amd.stream.engine import extend_condition
    Streams(monkeypatch)
    model = torch.nn.Module()
    model.cross = torch.nn.ModuleList([Layer(96, 40, 2) for _ in range(2)])
    ctx = paged.PagedContext(2, 3, 2, 48, 12, 'cpu', page_size=16, max_pages=20)
    ctx.resize(1, 20)
    seen = []

    def append(key, value, k, v, table, lengths, **how):
        seen.append((key.shape, ctx.lengths.tolist(), lengths.tolist(), table[0, :4].tolist()))
        if fails == 'layer' and len(seen) == 2:
            raise RuntimeError('the layer fails')
    monkeypatch.setattr(paged, 'paged_append', append)
    extend = lambda: extend_condition(model, ctx, 1, torch.zeros(1, 30, 41 if fails == 'width' else 40), torch.zeros(1, 30, 3))
    if fails:
        with pytest.raises(RuntimeError):
            extend()
        assert ctx.host_lengths == ctx.lengths.tolist() == [0, 20, 0]
        assert ctx._owned[1] == [0, 1] and ctx.free_pages == 10
    else:
        extend()
        assert ctx.host_lengths == ctx.lengths.tolist() == [0, 50, 0] and len(ctx._owned[1]) == 4
        assert [s[1:3] for s in seen] == [([0, 20, 0], [50])] * 2
        assert all(s[3] == ctx._owned[1] for s in seen)
    with pytest.raises(RuntimeError, match='pages left'):
        extend_condition(model, ctx, 1, torch.zeros(1, 200, 40), torch.zeros(1, 200, 3))
    with pytest.raises(ValueError, match='holds'):
        ctx.reserve(1, 10)


def test_a_tangent_goes_through_the_rotation(monkeypatch):
    """Forward mode, alone and over and under the gradient, with the launch replaced by the formula on the host: linear, so the
    tangent turns as x does. No tangent is dropped silently."""
    from torch.autograd import forward_ad as fw
    from streamvoxel_amd.stream import rotary as module

    def launch(x, out, positions, frequencies, layout, amplitude, inverse):
        angle = positions.double()[:, None] * frequencies
        c, s = amplitude * angle.cos(), (-1 if inverse else 1) * amplitude * angle.sin()
        a, b = x.double().chunk(2, -1)
        return out.copy_(torch.cat((a * c - b * s, b * c + a * s), -1))
    monkeypatch.setattr(module, '_launch', launch)
    monkeypatch.setattr(_lib, 'require_one_gpu', lambda *t: None)
    g = torch.Generator().manual_seed(3)
    x, t, dy = [torch.randn(2, 3, 5, 8, generator=g) for _ in range(3)]
    p, f = torch.arange(5) * 3, rotary_frequencies(8)[0]
    turn = lambda x: rotary(x, p, f, amplitude=1.5)
    want = turn(t)
    strange = t.transpose(2, 3).contiguous().transpose(2, 3)
    with fw.dual_level():
        for tangent in (t, strange):
            y = fw.unpack_dual(turn(fw.make_dual(x, tangent)))
            assert torch.equal(y.primal, turn(x)) and torch.equal(y.tangent, want)
        with torch.no_grad():
            assert torch.equal(fw.unpack_dual(turn(fw.make_dual(x, t))).tangent, want)
        leaf = x.clone().requires_grad_()
        y = fw.unpack_dual(turn(fw.make_dual(leaf, t)))
        assert torch.equal(y.tangent, want)
        back, = torch.autograd.grad(y.primal, leaf, dy)
        assert torch.equal(back, launch(dy, torch.empty_like(dy), p, f, 'half', 1.5, 1))
        # the tangent of the gradient: the transposed rotation of dy's
        leaf = x.clone().requires_grad_()
        back, = torch.autograd.grad(turn(leaf), leaf, fw.make_dual(dy, t), create_graph=True)
        assert torch.equal(fw.unpack_dual(back).tangent, launch(t, torch.empty_like(t), p, f, 'half', 1.5, 1))
        # the gradient of the tangent
        moving = t.clone().requires_grad_()
        tangent = fw.unpack_dual(turn(fw.make_dual(x, moving))).tangent
        back, = torch.autograd.grad(tangent, moving, dy)
        assert torch.equal(back, launch(dy, torch.empty_like(dy), p, f, 'half', 1.5, 1))
        with pytest.raises(ValueError, match='gradient'):
            rotary(fw.make_dual(x, t), p, f, out=torch.empty_like(x))
    assert torch.equal(turn(x), launch(x, torch.empty_like(x), p, f, 'half', 1.5, 0))


def test_strides_of_dimensions_with_one_element_are_not_looked_at(lib):
    """Rows are judged by the strides that a call uses: none for a dimension of one, or for the windows of packed tokens. (Calls
    that pass their checks up to a later one, or to the workspace's.)"""
    from streamvoxel_amd.stream.paged import _rows16
    error = lib.svhip_last_error
    assert append_call(lib, sk=(770, 68, 129)) == -1 and b'16-byte' in error()

    def attend(B=2, Hkv=2, N=3, pages=4, cu=0, sq=(768, 192, 64), so=(768, 192, 64), sk=(8192, 4096), m=20):
        cache = struct.pack('7P18q', FAKE, FAKE, 0, 0, FAKE, FAKE, 0, 1, B, Hkv, 64, pages, 64, m, m, *sk, 64, *sk, 64, 0, 0, 0, 0)
        args = struct.pack('4P10qd', FAKE, FAKE, cu, 0, 0, Hkv, N, *sq, *so, 0, 0.125)
        assert lib.svhip_paged_attention(cache, args, None) == -1
        return error()
    assert b'query rows' in attend(sq=(769, 192, 64)) and b'rows of out' in attend(so=(770, 192, 64))
    assert b'rows of a page' in attend(sk=(8193, 4096)) and b'rows of a page' in attend(sk=(8192, 4097))
    for kw in (dict(B=1, sq=(769, 192, 64), so=(770, 192, 64)), dict(Hkv=1, sq=(768, 193, 64), so=(768, 194, 64)),
               dict(N=1, sq=(768, 192, 65), so=(768, 192, 66)), dict(pages=1, sk=(8193, 4096)), dict(Hkv=1, sk=(8192, 4097)),
               dict(cu=FAKE, sq=(769, 192, 64), so=(770, 192, 64))):
        assert b'workspace' in attend(**kw), kw
    odd = torch.zeros(400, dtype=torch.bfloat16)
    for shape, strides in (((1, 2, 3, 8), (49, 24, 8, 1)), ((2, 1, 3, 8), (24, 7, 8, 1)), ((2, 3, 1, 8), (24, 8, 5, 1))):
        t = odd.as_strided(shape, strides)
        assert _rows16(t) is t
    for shape, strides in (((1, 2, 3, 8), (49, 24, 9, 1)), ((1, 1, 3, 8), (3, 5, 8, 1)), ((2, 3, 4, 8), (96, 32, 8, 1))):
        t = odd[1:].as_strided(shape, strides, 1)
        copy = _rows16(t)
        assert torch.equal(copy, t) and all(s % 8 == 0 for s in copy.stride()[:-1]) and copy.data_ptr() % 16 == 0


def test_an_append_has_a_place_for_every_row(monkeypatch):
    """Pages or exponents whose elements lie on each other, or keys and values in the same ones, would be written by two rows at
    once: refused before anything is launched. Halves of one buffer are places of their own."""
    from streamvoxel_amd.stream import paged
    launched = []
    monkeypatch.setattr(_lib, 'require_one_gpu', lambda *t: None)
    monkeypatch.setattr(_lib, 'launch', lambda *args: launched.append(args))
    x, n = torch.zeros(1, 2, 3, 8, dtype=torch.bfloat16), torch.ones(1, dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    both = torch.zeros(4, 2, 2, 16, 8, dtype=torch.bfloat16)
    codes, e = torch.zeros(2, 4, 2, 16, 8).to(torch.float8_e4m3fn), torch.zeros(2, 4, 2, 16, dtype=torch.uint8)
    append = lambda k, v, ke=None, ve=None: paged.paged_append(x, x, k, v, table, n, k_exponents=ke, v_exponents=ve)
    append(both[:, 0], both[:, 1])
    append(codes[0], codes[1], e[0], e[1])
    assert len(launched) == 2
    one = e[0, :1].expand(4, 2, 16)
    for args in ((both[:, 0], both[:, 0]), (both[:1, 0].expand(4, 2, 16, 8), both[:, 1]), (codes[0], codes[0], e[0], e[1]),
                 (codes[0], codes[1], e[0], e[0]), (codes[0], codes[1], one, e[1]), (codes[0], codes[1], e[1], one)):
        with pytest.raises(ValueError, match='place|share'):
            append(*args)
    assert len(launched) == 2


def test_a_capture_does_not_change_the_books(monkeypatch):
    """What a capture would send is a host number of that moment, which every replay would send again: refused, and nothing
    changes."""
    from streamvoxel_amd.stream.paged import PagedContext
    stream, capturing = RecordedStream('main'), [False]
    monkeypatch.setattr(PagedContext, '_stream', lambda self: stream)
    monkeypatch.setattr(PagedContext, '_capturing', lambda self: capturing[0], raising=False)
    monkeypatch.setattr(PagedContext, '_send', staticmethod(lambda to, v: to.copy_(torch.tensor(v, dtype=torch.int32))))
    ctx = PagedContext(1, 2, 2, 64, 6, 'cpu', page_size=16)
    ctx.grow(20)
    capturing[0] = True
    for change in (lambda: ctx.grow(1), lambda: ctx.grow(20), lambda: ctx.release(1), lambda: ctx.resize(0, 0),
                   lambda: ctx.reserve(1, 60)):
        with pytest.raises(RuntimeError, match='capture'):
            change()
        assert ctx.lengths.tolist() == ctx.host_lengths == [20, 20] and ctx._owned == [[0, 1], [2, 3]]
        assert ctx.free_pages == 2 and not stream.work
    capturing[0] = False
    ctx.grow(1)
    assert ctx.lengths.tolist() == [21, 21]


def test_an_append_to_pages_without_heads_or_of_no_pool_writes_nothing(monkeypatch):
    """Empty pools share the null address and nothing else: not refused for it."""
    from streamvoxel_amd.stream import paged
    launched = []
    monkeypatch.setattr(_lib, 'require_one_gpu', lambda *t: None)
    monkeypatch.setattr(_lib, 'launch', lambda *args: launched.append(args))
    n, table = torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    for shape in ((4, 0, 16, 8), (0, 2, 16, 8)):
        k, v = [torch.zeros(shape, dtype=torch.bfloat16) for _ in 'kv']
        x = torch.zeros(1, shape[1], 3, 8, dtype=torch.bfloat16)
        paged.paged_append(x, x, k, v, table, n)
    assert len(launched) == 2
