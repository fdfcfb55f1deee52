"""Normed and rotated queries and keys on the GPU, against plain float64 on the host and against differences.

Tolerances. A row's unit x / sqrt(mean x^2 + eps) is off by half of what its sum of squares is, relatively: a lane adds 16
squares and 5 steps add the lanes', 21 * 2^-24 and 2^-24 for each product, so 11 * 2^-24; by 2 * 2^-24 for the square root's
reciprocal and 2 * 2^-24 for mean and eps; the products with unit and weight add 2 * 2^-24: 17 * 2^-24. The rotation is off by
8 * 2^-24 of |a| + |b| of its pair (test_gpu_rotary.py). So a result is off by 25 * 2^-24 of what its pair's magnitudes add up
to, and half a step of its type.
Gradient, with G the pair's |dy_a| + |dy_b| times the amplitude: c = w g is off by 9 * 2^-24 |w| G; mean(c u) sums 256 such products at
most, off by (9 + 17 + 22) * 2^-24 of the mean of |w| G |u|; unit and its products add 17 + 3 more of each term.
Weights: each term g u is off by (8 + 17) * 2^-24 G |u|, and the sum by 2^-24 for each addition on a term's way: those of its lane
(rows / 8 at most: 8 rows at once), 10 in the workgroup and 64 over the workgroups."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
E = 2.0 ** -24


def _case(msg):
    print(f'[gpu-case] {msg}', flush=True)


def half_step(t):
    return torch.finfo(t.dtype).eps / 2


def turn64(x, positions, freq, layout, sign=1.0):
    """x [B, H, N, D] float64 turned; positions [B, N]."""
    half = len(freq)
    angle = positions.double()[:, None, :, None] * freq
    c, s = angle.cos(), sign * angle.sin()
    y = x.clone()
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == 'half' else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def pair_sum(x, half, layout):
    """|a| + |b| of each element's pair; twice the magnitude of one that is kept."""
    y = 2 * x.abs()
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == 'half' else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    y[..., a] = y[..., b] = x[..., a].abs() + x[..., b].abs()
    return y


def reference(x, w, positions, freq, layout, amplitude, eps, dy=None):
    """{what: (value, allowed error before the result's own rounding)} in float64, on the host."""
    x, half = x.double().cpu(), len(freq)
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double().cpu()
    D = x.shape[-1]
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    u = x * r
    scale = torch.ones(D, dtype=torch.float64)
    scale[:2 * half] = amplitude
    out = dict(y=(turn64(u * w, positions, freq, layout) * scale, 25 * E * pair_sum(u * w, half, layout) * scale.abs()))
    if dy is None:
        return out
    dy = dy.double().cpu()
    g, G = turn64(dy * scale, positions, freq, layout, -1.0), pair_sum(dy * scale, half, layout)
    c, C = g * w, G * w.abs()
    dot = (c * u).mean(-1, keepdim=True)
    mean = (C * u.abs()).mean(-1, keepdim=True)
    out['dx'] = (r * (c - u * dot), E * r * (29 * C + u.abs() * 68 * mean))
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    out['dw'] = ((g * u).sum((0, 1, 2)), (25 + 74 + rows / 8) * E * (G * u.abs()).sum((0, 1, 2)))
    return out


def check(got, expected, what):
    value, err = expected
    off = (got.detach().cpu().double() - value).abs()
    assert not torch.isnan(off).any(), what
    allowed = err + half_step(got) * (value.abs() + err) + 1e-37
    assert (off <= allowed).all(), (what, (off / allowed).max().item())


def inputs(B, N, H, Hk, D, dtype, wdtype, seed, fused=True):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(B, N, H + Hk, D, generator=g).to(dtype).to(DEV)
    q, k = rows[:, :, :H].transpose(1, 2), rows[:, :, H:].transpose(1, 2)
    if not fused:
        q, k = q.contiguous(), k.contiguous()
    weights = [(1 + 0.3 * torch.randn(D, generator=g)).to(wdtype).to(DEV) for _ in 'qk']
    dy = [torch.randn(B, N, n, D, generator=g).to(dtype).to(DEV).transpose(1, 2) for n in (H, Hk)]
    return q, k, *weights, *dy


SHAPES = [(1, 1, 1, 1, 64, 32), (2, 7, 4, 2, 64, 32), (3, 1, 12, 12, 48, 24), (1, 33, 5, 1, 96, 16), (2, 65, 8, 2, 128, 64),
          (1, 9, 2, 3, 256, 128), (2, 5, 3, 1, 200, 8), (1, 600, 2, 1, 80, 40)]
ODD = [(2, 5, 3, 2, 2, 1), (1, 19, 4, 1, 7, 2), (2, 6, 2, 2, 36, 18), (1, 8, 2, 1, 64, 1), (1, 3, 1, 1, 255, 120), (2, 4, 3, 1, 72, 12),
       (1, 5, 2, 2, 17, 8)]


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('dtype, wdtype', [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.float32, torch.float32)], ids=str)
@pytest.mark.parametrize('shape', SHAPES + ODD, ids=str)
def test_results_and_gradients_against_float64(shape, dtype, wdtype, layout):
    from streamvoxel_amd.stream.rotary import norm_rotary
    B, N, H, Hk, D, half = shape
    _case(f'norm_rotary {shape} {dtype} {wdtype} {layout}')
    q, k, wq, wk, dq, dk = inputs(B, N, H, Hk, D, dtype, wdtype, D + N)
    g = torch.Generator().manual_seed(1)
    positions = torch.randint(-50, 200000, (B, N), generator=g)
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    amplitude, eps = 1.25, 1e-5
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = norm_rotary(*leaves, positions.to(DEV), freq.to(DEV), eps=eps, layout=layout, amplitude=amplitude)
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    plain = norm_rotary(q, k, wq, wk, positions.to(DEV).int(), freq.to(DEV), eps=eps, layout=layout, amplitude=amplitude)
    assert torch.equal(plain[0], yq) and torch.equal(plain[1], yk) and not plain[0].requires_grad
    for i, (x, w, dy, y) in enumerate(((q, wq, dq, yq), (k, wk, dk, yk))):
        ref = reference(x, w, positions, freq, layout, amplitude, eps, dy)
        check(y, ref['y'], 'y')
        check(grads[i], ref['dx'], 'dx')
        check(grads[2 + i], ref['dw'], 'dw')
        assert grads[i].dtype == dtype and grads[2 + i].dtype == wdtype


def test_gradient_against_differences():
    """fp32, the loss a fixed sum: central differences of the plain formula in float64 along a random direction of each leaf."""
    from streamvoxel_amd.stream.rotary import norm_rotary
    B, N, H, Hk, D, half = 2, 6, 3, 2, 48, 20
    leaves = inputs(B, N, H, Hk, D, torch.float32, torch.float32, 5)
    q, k, wq, wk, dq, dk = leaves
    positions = torch.arange(N)[None] + torch.tensor([[3], [100]])
    freq = 1000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    params = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = norm_rotary(*params, positions.to(DEV), freq.to(DEV), layout='half')
    grads = torch.autograd.grad(out, params, (dq, dk))

    def loss(ts):
        total = 0.0
        for x, w, dy in ((ts[0], ts[2], dq), (ts[1], ts[3], dk)):
            u = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
            total += (turn64(u * w, positions, freq, 'half') * dy.cpu().double()).sum()
        return total

    base = [t.detach().cpu().double() for t in (q, k, wq, wk)]
    g = torch.Generator().manual_seed(9)
    for i, grad in enumerate(grads):
        direction = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        h = 1e-4
        moved = [[t + s * h * direction if j == i else t for j, t in enumerate(base)] for s in (1, -1)]
        slope = (loss(moved[0]) - loss(moved[1])) / (2 * h)
        along = (grad.cpu().double() * direction).sum()
        # (The difference's own error is h^2 / 6 of a third derivative, 2e-9 times the magnitudes' sum; the gradient's, above.)
        assert abs(along - slope) <= 1e-5 * (grad.cpu().double().abs() * direction.abs()).sum()


@pytest.mark.parametrize('missing', ['weights', 'key', 'one weight'])
def test_parts_that_may_be_missing(missing):
    from streamvoxel_amd.stream.rotary import norm_rotary
    q, k, wq, wk, dq, dk = inputs(2, 11, 4, 2, 64, torch.bfloat16, torch.bfloat16, 3)
    positions, freq = torch.arange(11), 100.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    if missing == 'key':
        k = wk = None
    elif missing == 'weights':
        wq = wk = None
    else:
        wk = None
    leaves = [None if t is None else t.detach().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = norm_rotary(*leaves, positions.to(DEV), freq.to(DEV))
    assert (yk is None) == (missing == 'key')
    outs = [y for y in (yq, yk) if y is not None]
    grads = torch.autograd.grad(outs, [t for t in leaves if t is not None], [dq, dk][:len(outs)])
    there = [i for i, t in enumerate(leaves) if t is not None]
    for i, y in enumerate(outs):
        ref = reference((q, k)[i], (wq, wk)[i], positions[None].expand(2, -1), freq, 'half', 1.0, 1e-6, (dq, dk)[i])
        check(y, ref['y'], 'y')
        check(grads[there.index(i)], ref['dx'], 'dx')
        if leaves[2 + i] is not None:
            check(grads[there.index(2 + i)], ref['dw'], 'dw')


def test_some_leaves_alone_and_a_result_that_is_not_used():
    from streamvoxel_amd.stream.rotary import norm_rotary
    q, k, wq, wk, dq, dk = inputs(2, 30, 4, 4, 64, torch.float32, torch.float32, 3)
    positions, freq = torch.arange(30, device=DEV), (100.0 ** (-torch.arange(16, dtype=torch.float64) / 16)).to(DEV)
    every = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    full = torch.autograd.grad(norm_rotary(*every, positions, freq), every, (dq, dk))
    for which in range(4):
        leaves = [t.detach() for t in (q, k, wq, wk)]
        leaves[which].requires_grad_()
        out = norm_rotary(*leaves, positions, freq)
        assert torch.equal(torch.autograd.grad(out, leaves[which], (dq, dk))[0], full[which])
    out = norm_rotary(*every, positions, freq)[1]
    got = torch.autograd.grad(out, every, dk)
    assert not got[0].any() and not got[2].any() and torch.equal(got[1], full[1]) and torch.equal(got[3], full[3])


def test_broadcast_gradients_and_views():
    """A gradient expanded over tokens, odd strides, rows off their 16-byte alignment, a gradient whose head_dim is not
    contiguous."""
    from streamvoxel_amd.stream.rotary import norm_rotary
    g = torch.Generator().manual_seed(4)
    big = torch.randn(2, 9, 3, 75, generator=g).to(torch.bfloat16).to(DEV)
    q, k = big[..., 1:65].transpose(1, 2), big[:, ::1, 1:, 3:67].transpose(1, 2)
    w = torch.rand(64, generator=g).to(DEV)
    freq = (50.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).to(DEV)
    positions = torch.arange(9, device=DEV)
    dq = torch.randn(2, 3, 1, 64, generator=g).to(torch.bfloat16).to(DEV).expand(2, 3, 9, 64)
    dk = torch.randn(2, 2, 64, 9, generator=g).to(torch.bfloat16).to(DEV).transpose(2, 3)
    leaves = [t.detach().requires_grad_() for t in (q, k, w)]
    out = norm_rotary(leaves[0], leaves[1], leaves[2], leaves[2], positions, freq)
    grads = torch.autograd.grad(out, leaves, (dq, dk))
    refs = [reference(x, w, positions.cpu()[None].expand(2, -1), freq.cpu(), 'half', 1.0, 1e-6, dy)
            for x, dy in ((q, dq), (k, dk))]
    for i in (0, 1):
        check(out[i], refs[i]['y'], 'y')
        check(grads[i], refs[i]['dx'], 'dx')
    both = refs[0]['dw'][0] + refs[1]['dw'][0], refs[0]['dw'][1] + refs[1]['dw'][1] + 2 * E * (
        refs[0]['dw'][0].abs() + refs[1]['dw'][0].abs())
    check(grads[2], both, 'dw of a shared weight')


@pytest.mark.parametrize('step', [1, 5, 64])
def test_rows_that_overlap(step):
    """Queries and keys as windows that slide over one sequence, `step` elements a token, and the same rows rotated alone."""
    from streamvoxel_amd.stream.rotary import norm_rotary, rotary
    g = torch.Generator().manual_seed(step)
    line = torch.randn(2, 3, 6 * step + 64, generator=g).to(torch.bfloat16).to(DEV)
    q, k = line.unfold(2, 64, step), line[:, :2].unfold(2, 64, step)
    w = (1 + 0.3 * torch.randn(64, generator=g)).to(DEV)
    positions, freq = torch.arange(7), 50.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    dy = [torch.randn(t.shape, generator=g).to(torch.bfloat16).to(DEV) for t in (q, k)]
    leaves = [t.detach().requires_grad_() for t in (q, k, w)]
    out = norm_rotary(leaves[0], leaves[1], leaves[2], None, positions.to(DEV), freq.to(DEV))
    plain = norm_rotary(q, k, w, None, positions.to(DEV), freq.to(DEV))
    grads = torch.autograd.grad(out, leaves, dy)
    for i, (x, weight) in enumerate(((q, w), (k, None))):
        ref = reference(x, weight, positions[None].expand(2, -1), freq, 'half', 1.0, 1e-6, dy[i])
        check(out[i], ref['y'], 'y')
        check(grads[i], ref['dx'], 'dx')
        assert torch.equal(out[i], plain[i])
        if i == 0:
            check(grads[2], ref['dw'], 'dw')
    rows, pairs = q.double().cpu(), pair_sum(q.double().cpu(), 32, 'half')
    check(rotary(q, positions.to(DEV), freq.to(DEV)), (turn64(rows, positions[None], freq, 'half'), 8 * E * pairs), 'rotary')


def test_in_place_in_the_projection_and_refused_places():
    from streamvoxel_amd.stream.rotary import norm_rotary
    q, k, wq, wk, *_ = inputs(2, 10, 4, 2, 64, torch.bfloat16, torch.bfloat16, 8)
    positions, freq = torch.arange(10, device=DEV), (50.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).to(DEV)
    want = norm_rotary(q, k, wq, wk, positions, freq)
    both = torch.empty_like(q)
    for out, what in (((k.new_empty(2, 4, 10, 64), q[:, 1:3]), 'memory'), ((both, both[:, :2]), 'memory'),
                      ((q.new_empty(2, 1, 10, 64).expand(2, 4, 10, 64), torch.empty_like(k)), 'place'),
                      ((both, None), 'pair'), ((k, torch.empty_like(k)), 'shape')):
        with pytest.raises(ValueError, match=what):
            norm_rotary(q, k, wq, wk, positions, freq, out=out)
    leaf = q.detach().requires_grad_()
    with pytest.raises(ValueError, match='gradient'):
        norm_rotary(leaf, k, wq, wk, positions, freq, out=(torch.empty_like(q), torch.empty_like(k)))
    got = norm_rotary(q, k, wq, wk, positions, freq, out=(q, k))
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_infinities_and_nan_stay_in_their_rows_and_zeros_give_zeros():
    from streamvoxel_amd.stream.rotary import norm_rotary
    q, k, wq, wk, dq, dk = inputs(1, 8, 4, 2, 72, torch.float32, torch.float32, 2, fused=False)
    positions, freq = torch.arange(8, device=DEV), (50.0 ** (-torch.arange(33, dtype=torch.float64) / 33)).to(DEV)
    want = norm_rotary(q, k, wq, wk, positions, freq)
    q[0, 1, 3, 5], q[0, 2, 0, 71], k[0, 0, 4, 0] = math.nan, math.inf, -math.inf
    q[0, 3, 7] = 0.0
    got = norm_rotary(q, k, wq, wk, positions, freq)
    ok = torch.ones(1, 4, 8, dtype=torch.bool, device=DEV)
    ok[0, 1, 3] = ok[0, 2, 0] = ok[0, 3, 7] = False
    assert torch.equal(got[0][ok], want[0][ok]) and got[0][0, 1, 3].isnan().all() and got[0][0, 2, 0].isnan().any()
    assert not got[0][0, 3, 7].any() and got[1][0, 0, 4].isnan().any() and torch.equal(got[1][0, 1], want[1][0, 1])
    leaf = q.detach().requires_grad_()
    dx = torch.autograd.grad(norm_rotary(leaf, k, wq, wk, positions, freq)[0], leaf, dq)[0]
    assert dx[0, 3, 7].isfinite().all() and dx[0, 0].isfinite().all()


def test_the_same_bits_from_call_to_call_on_a_stream_and_in_a_graph():
    """Eager, on another stream, and captured with its gradient: several replays with other inputs between them."""
    from streamvoxel_amd.stream.rotary import norm_rotary
    q, k, wq, wk, dq, dk = inputs(2, 700, 8, 2, 128, torch.bfloat16, torch.float32, 6)
    positions, freq = torch.arange(700, device=DEV), (1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)).to(DEV)

    def step(*leaves):
        y = norm_rotary(*leaves, positions, freq)
        return *[t.detach() for t in y], *torch.autograd.grad(y, leaves, (dq, dk))

    fresh = lambda: [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    want = step(*fresh())
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(*fresh()), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = fresh()
        got = step(*leaves)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            static = step(*leaves)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.Generator().manual_seed(7)
    for _ in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=g).to(q.dtype))
            wq.copy_(torch.rand(128, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        again = step(*fresh())
        assert all(torch.equal(a, b) for a, b in zip(static, again))
        (q.float() @ q.float().transpose(2, 3)).sum()


@pytest.mark.parametrize('sizes', [(0, 3, 2, 1), (2, 0, 2, 1), (2, 3, 0, 1), (2, 3, 2, 0)], ids=str)
def test_empty_batches(sizes):
    from streamvoxel_amd.stream.rotary import norm_rotary
    B, N, H, Hk = sizes
    q, k, wq, wk, dq, dk = inputs(B, N, H, Hk, 64, torch.bfloat16, torch.float32, 1)
    positions, freq = torch.arange(N, device=DEV), (50.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).to(DEV)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    y = norm_rotary(*leaves, positions, freq)
    assert y[0].shape == q.shape and y[1].shape == k.shape
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    if B * N * H == 0:
        assert not grads[2].any()
    if B * N * Hk == 0:
        assert not grads[3].any()


def test_refusals():
    from streamvoxel_amd.stream.rotary import norm_rotary
    q, k, wq, wk, dq, dk = inputs(1, 4, 2, 2, 64, torch.bfloat16, torch.float32, 1)
    p, f = torch.arange(4, device=DEV), torch.ones(32, dtype=torch.float64, device=DEV)
    for args, error in (((q.half(), k.half(), wq, wk, p, f), TypeError), ((q, k.float(), wq, wk, p, f), TypeError),
                        ((q, k, wq, wk.bfloat16(), p, f), TypeError), ((q, k, wq[:32], wk, p, f), ValueError),
                        ((q, k[:, :, :3], wq, wk, p, f), ValueError), ((q, None, wq, wk, p, f), ValueError),
                        ((q, k, wq, wk, p.float(), f), ValueError), ((q, k, wq, wk, p, f.float()), ValueError),
                        ((q, k, wq, wk, p, torch.ones(33, dtype=torch.float64, device=DEV)), ValueError),
                        ((q.transpose(2, 3), k, wq, wk, p, f), ValueError), ((q[0], k, wq, wk, p, f), ValueError),
                        ((q, k, wq, wk, p.cpu(), f), RuntimeError)):
        with pytest.raises(error):
            norm_rotary(*args)
    for eps in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match='eps'):
            norm_rotary(q, k, wq, wk, p, f, eps=eps)
    with pytest.raises(ValueError, match='layout'):
        norm_rotary(q, k, wq, wk, p, f, layout='axial')
    wide = torch.zeros(1, 1, 4, 264, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match='head_dim'):
        norm_rotary(wide, None, None, None, p, f)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):      # no tangent is dropped
        norm_rotary(fwd.make_dual(q, torch.ones_like(q)), k, wq, wk, p, f)
    leaf = q.float().detach().requires_grad_()
    y = norm_rotary(leaf, None, None, None, p, f)[0]
    dx = torch.autograd.grad(y, leaf, torch.ones_like(y).requires_grad_(), create_graph=True)[0]
    with pytest.raises(RuntimeError):      # once differentiable
        torch.autograd.grad(dx.sum(), leaf)


def test_more_tokens_than_one_launch_holds():
    """8.4 million windows of one token: past the workgroups of one launch."""
    from streamvoxel_amd.stream.rotary import norm_rotary
    B = (1 << 23) + 5
    x = torch.ones(B, 1, 1, 8, dtype=torch.bfloat16, device=DEV)
    x[-3:, :, :, 0] = 3.0
    f = torch.ones(4, dtype=torch.float64, device=DEV)
    y = norm_rotary(x, None, None, None, torch.zeros(1, dtype=torch.int32, device=DEV), f)[0]
    assert (y[:-3] == 1).all()
    want = torch.ones(8, dtype=torch.float64)
    want[0] = 3.0
    check(y[-3:].reshape(3, 8), (want / (want.pow(2).mean() + 1e-6).sqrt(), 25 * E * want), 'last rows')
