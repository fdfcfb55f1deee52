"""Rotary positions on the GPU against their formula in 64 bits, and the gradient against the formula's and differences.

Tolerance: cos and sin are off by at most half a step of the fp32 half-turns (pi 2^-25), 2 steps of sincospi and the
amplitude's rounding, 6 * 2^-24 in all, the two products and the sum by 2 * 2^-24 more: 8 * 2^-24 of A (|x_a| + |x_b|),
and half a step of the type (torch.finfo(type).eps / 2 of the result) when it is rounded."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def pairs_of(half, layout):
    i = torch.arange(half)
    return (i, i + half) if layout == 'half' else (2 * i, 2 * i + 1)


def formula(x, positions, freq, layout, amplitude=1.0, sign=1.0):
    """(y, allowed error before rounding) in float64 on the host; positions [B, N]."""
    x, freq = x.detach().cpu().double(), freq.cpu()
    angle = (positions.cpu().double()[..., None] * freq)[:, None]
    c, s = amplitude * angle.cos(), sign * amplitude * angle.sin()
    a, b = pairs_of(freq.numel(), layout)
    y, err = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    err[..., a] = err[..., b] = 8 * 2.0 ** -24 * abs(amplitude) * (x[..., a].abs() + x[..., b].abs())
    return y, err


def check(got, x, positions, freq, layout, amplitude=1.0, sign=1.0):
    y, err = formula(x, positions, freq, layout, amplitude, sign)
    err = err + torch.finfo(got.dtype).eps / 2 * (y.abs() + err)
    kept = freq.numel() * 2
    err[..., kept:] = 0
    assert got.dtype == x.dtype and got.shape == x.shape
    off = (got.detach().cpu().double() - y).abs() - err
    assert off.max().item() <= 0, off.max().item()


def freqs(pairs):
    return (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).to(DEV)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('shape, part', [((1, 1, 1, 2), 2), ((2, 3, 5, 64), 64), ((3, 12, 17, 64), 32), ((1, 4, 1, 128), 96),
                                         ((2, 5, 9, 38), 38), ((1, 2, 33, 110), 62), ((1, 1, 1025, 256), 256),
                                         ((64, 8, 1, 96), 96), ((1, 33, 8, 24), 4), ((2, 2, 7, 20), 8),
                                         ((1, 3, 4, 300), 200)])
def test_rotary_against_the_formula(shape, part, layout, dtype):
    from streamvoxel_amd.stream.rotary import rotary
    g = torch.Generator().manual_seed(sum(shape) + part)
    B, H, N, D = shape
    x = torch.randn(B, N, H, D, generator=g).to(dtype).to(DEV).transpose(1, 2)
    positions = torch.randint(-50, 100000, (B, N), generator=g).to(DEV)
    check(rotary(x, positions, freqs(part // 2), layout, 1.25), x, positions, freqs(part // 2), layout, 1.25)
    dense, shared = x.contiguous(), positions[0].to(torch.int32)
    check(rotary(dense, shared, freqs(part // 2), layout), x, shared.expand(B, N), freqs(part // 2), layout)
    inplace = dense.clone()
    assert rotary(inplace, positions, freqs(part // 2), layout, out=inplace) is inplace
    assert torch.equal(inplace, rotary(dense, positions, freqs(part // 2), layout))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_rotary_of_views_in_odd_places(dtype):
    from streamvoxel_amd.stream.rotary import rotary
    g = torch.Generator().manual_seed(5)
    buffer = torch.randn(3, 11, 2, 5, 67, generator=g).to(dtype).to(DEV)
    positions = torch.randint(0, 4000, (3, 22), generator=g).to(DEV)[:, ::2]
    for x in (buffer[:, :, 1, :, 1:65], buffer[:, :, 0, ::2, 3:67], buffer[:, :, 1, :, :64]):
        x = x.transpose(1, 2)
        check(rotary(x, positions, freqs(32), 'half'), x, positions, freqs(32), 'half')
        out = torch.full((3, 11, x.shape[1], 66), 7.0, dtype=dtype, device=DEV)
        rotary(x, positions, freqs(32), 'interleaved', out=out[..., 1:65].transpose(1, 2))
        check(out[..., 1:65].transpose(1, 2), x, positions, freqs(32), 'interleaved')
        assert (out[..., 0] == 7).all() and (out[..., 65] == 7).all()


def test_rotary_keeps_the_angle_of_far_positions():
    from streamvoxel_amd.stream.rotary import rotary
    x = torch.randn(1, 2, 6, 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    for far in (1 << 20, (1 << 30) - 8, -(1 << 30)):
        positions = far + torch.arange(6, device=DEV)[None]
        check(rotary(x, positions, freqs(32), 'half'), x, positions, freqs(32), 'half')


def test_rotary_with_no_tokens_heads_or_windows():
    from streamvoxel_amd.stream.rotary import rotary
    for shape in ((0, 2, 3, 8), (2, 0, 3, 8), (2, 2, 0, 8)):
        x = torch.zeros(shape, device=DEV)
        y = rotary(x, torch.zeros(shape[0], shape[2], dtype=torch.int32, device=DEV), freqs(4))
        assert y.shape == x.shape


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_rotary_gradient_is_the_transposed_rotation(layout, dtype):
    from streamvoxel_amd.stream.rotary import rotary
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 3, 10, 48, generator=g).to(dtype).to(DEV).requires_grad_()
    dy = torch.randn(2, 10, 3, 48, generator=g).to(dtype).to(DEV).transpose(1, 2)
    positions = torch.randint(0, 9000, (2, 10), generator=g).to(DEV)
    y = rotary(x, positions, freqs(20), layout, 1.1)
    check(y, x, positions, freqs(20), layout, 1.1)
    y.backward(dy)
    check(x.grad, dy, positions, freqs(20), layout, 1.1, sign=-1.0)
    x.grad = None
    rotary(x, positions, freqs(20), layout).sum().backward()       # an expanded gradient
    check(x.grad, torch.ones_like(dy), positions, freqs(20), layout, sign=-1.0)


def test_rotary_gradient_against_differences():
    """A linear map: the difference over any step is the derivative, off by the fp32 errors of the two values alone."""
    from streamvoxel_amd.stream.rotary import rotary
    g = torch.Generator().manual_seed(9)
    x = torch.randn(1, 2, 3, 16, generator=g).to(DEV).requires_grad_()
    w = torch.randn(1, 2, 3, 16, generator=g).to(DEV)
    positions = torch.tensor([[3, 70, 900]], device=DEV)
    loss = lambda t: (rotary(t, positions, freqs(6), 'half').double() * w.double()).sum()
    loss(x).backward()
    with torch.no_grad():
        for i in range(0, x.numel(), 5):
            step = torch.zeros(x.numel(), device=DEV)
            step[i] = 2.0
            moved = x + step.view_as(x)
            difference = (loss(moved) - loss(x)).item() / (moved - x).double().sum().item()
            # Each value: 8 * 2^-24 (|x_a| + |x_b|) and its rounding (2^-24 of it) times |w|, over both and the step of 2.
            bound = 2.0 ** -24 * 10 * ((moved.abs() + x.abs()).double().sum() * w.abs().max().double()).item()
            assert abs(difference - x.grad.view(-1)[i].item()) <= bound


def test_rotary_in_a_graph_replays_with_new_contents():
    from streamvoxel_amd.stream.rotary import rotary
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 4, 6, 64, generator=g).to(torch.bfloat16).to(DEV)
    positions = torch.arange(6, dtype=torch.int32, device=DEV)
    f = freqs(32)
    rotary(x, positions, f)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotary(x, positions, f)
    for step in range(4):
        x.copy_(torch.randn(2, 4, 6, 64, generator=g).to(torch.bfloat16))
        positions.add_(17 * step)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, rotary(x, positions, f))


def test_rotary_refuses_on_the_gpu():
    from streamvoxel_amd.stream.rotary import rotary
    x, p, f = torch.zeros(1, 2, 3, 8, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV), freqs(4)
    for bad in (lambda: rotary(x, p, f, 'axial'), lambda: rotary(x, p.float(), f), lambda: rotary(x, p[:2], f),
                lambda: rotary(x, p, f.float()), lambda: rotary(x, p, freqs(5)), lambda: rotary(x[0], p, f),
                lambda: rotary(x.transpose(2, 3), p, f), lambda: rotary(x, p, f, out=x[:, :, :, :4]),
                lambda: rotary(x, p, f, out=x.flatten()[:48].view(1, 2, 3, 8).flip(1).contiguous()[:, :1]),
                lambda: rotary(x.requires_grad_(), p, f, out=torch.empty_like(x))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        rotary(torch.zeros(1, 2, 3, 8, dtype=torch.float16, device=DEV), p, f)
    buffer = torch.zeros(1, 2, 4, 8, device=DEV)
    with pytest.raises(ValueError, match='share'):
        rotary(buffer[:, :, :3], p, f, out=buffer[:, :, 1:])
    with pytest.raises(ValueError, match='place'):
        rotary(buffer[:, :, :3].clone(), p, f, out=torch.zeros(1, 1, 3, 8, device=DEV).expand(1, 2, 3, 8))


def test_rotary_gradient_in_a_graph():
    from streamvoxel_amd.stream.rotary import rotary
    g = torch.Generator().manual_seed(8)
    x = torch.randn(2, 3, 50, 64, generator=g).to(DEV).requires_grad_()
    dy, positions, f = torch.randn(2, 3, 50, 64, generator=g).to(DEV), torch.arange(50, device=DEV), freqs(32)
    rotary(x.detach(), positions, f)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotary(x, positions, f, 'interleaved')
        dx, = torch.autograd.grad(y, x, dy)
    for step in range(3):
        dy.copy_(torch.randn(2, 3, 50, 64, generator=g))
        positions.add_(5 * step)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.detach(), rotary(x.detach(), positions, f, 'interleaved'))
        # The transposed rotation is the rotation by the negative angle, whose sines are the same numbers negated.
        assert torch.equal(dx, rotary(dy, -positions, f, 'interleaved'))


def test_rotary_gradient_of_the_gradient():
    """The rotation is linear: the gradient of <w, dx> by dy is the rotation of w, whatever the order."""
    from streamvoxel_amd.stream.rotary import rotary
    g = torch.Generator().manual_seed(9)
    x, w = [torch.randn(2, 3, 20, 32, generator=g).to(DEV) for _ in 'xw']
    dy = torch.randn(2, 3, 20, 32, generator=g).to(DEV).requires_grad_()
    positions, f = torch.arange(20, device=DEV) * 7, freqs(16)
    y = rotary(x.requires_grad_(), positions, f, amplitude=1.5)
    dx, = torch.autograd.grad(y, x, dy, create_graph=True)
    ddy, = torch.autograd.grad(dx, dy, w, create_graph=True)
    assert torch.equal(ddy.detach(), rotary(w, positions, f, amplitude=1.5))
    again, = torch.autograd.grad(y, x, dy.detach())
    assert torch.equal(again, dx.detach())


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_rotary_in_forward_mode(layout, dtype):
    """A linear map: the tangent of the result is the rotation of x's tangent, of a leaf's too."""
    from torch.autograd import forward_ad as fw
    from streamvoxel_amd.stream.rotary import rotary
    g = torch.Generator().manual_seed(12)
    x, t = [torch.randn(2, 9, 3, 40, generator=g).to(dtype).to(DEV).transpose(1, 2) for _ in range(2)]
    positions, f = torch.randint(0, 9000, (2, 9), generator=g).to(DEV), freqs(16)
    with fw.dual_level():
        for leaf in (x, x.clone().requires_grad_()):
            y = fw.unpack_dual(rotary(fw.make_dual(leaf, t), positions, f, layout, 1.5))
            check(y.primal, x, positions, f, layout, 1.5)
            check(y.tangent, t, positions, f, layout, 1.5)
        with pytest.raises(ValueError, match='gradient'):
            rotary(fw.make_dual(x, t), positions, f, out=torch.empty_like(x))


def test_rotary_of_more_windows_than_one_launch_holds():
    """More than 2^24 workgroups, which no launch of 256 threads each holds; against the formula on the GPU."""
    from streamvoxel_amd.stream.rotary import rotary
    B = (1 << 24) + 5
    x = torch.randn(B, 1, 1, 8, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    positions = torch.arange(B, dtype=torch.int32, device=DEV)[:, None]
    f = freqs(4)
    got = rotary(x, positions, f)
    for at in range(0, B, 1 << 22):
        cut = slice(at, at + (1 << 22))
        angle = (positions[cut].double() * f)[:, None, None]
        a, b = x[cut].double().chunk(2, -1)
        y = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)
        err = 8 * 2.0 ** -24 * (a.abs() + b.abs()).repeat(1, 1, 1, 2)
        assert ((got[cut].double() - y).abs() <= err + 2.0 ** -24 * (y.abs() + err)).all(), at
