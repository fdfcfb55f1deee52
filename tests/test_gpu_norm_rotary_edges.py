"""norm_rotary on the GPU at sizes and values out of the ordinary, against plain float64 on the host: an eps that fp32 does not
hold.

Tolerances: those of test_gpu_norm_rotary.py."""
import pytest
import torch

from test_gpu_norm_rotary import check, inputs, reference

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def _case(msg):
    print(f'[gpu-case] {msg}', flush=True)


@pytest.mark.parametrize('eps', [1e-50, 1e-44, 1e-40, 1e-300])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=str)
def test_rows_of_zeros_at_the_least_eps(dtype, eps):
    from streamvoxel_amd.stream.rotary import norm_rotary
    q, k, wq, wk, dq, dk = inputs(1, 8, 4, 2, 64, dtype, torch.float32, 2, fused=False)
    q[0, 1, 3], k[0, 0] = 0.0, 0.0
    positions, freq = torch.arange(8), 50.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    got = norm_rotary(q, k, wq, wk, positions.to(DEV), freq.to(DEV), eps=eps)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        check(y, reference(x, w, positions[None], freq, 'half', 1.0, eps)['y'], 'y')
    assert not got[0][0, 1, 3].any() and not got[1][0, 0].any()
    leaf = q.detach().requires_grad_()
    dx = torch.autograd.grad(norm_rotary(leaf, k, wq, wk, positions.to(DEV), freq.to(DEV), eps=eps)[0], leaf, dq)[0]
    others = torch.ones(4, 8, dtype=torch.bool, device=DEV)
    others[1, 3] = False
    assert dx[0][others].isfinite().all() and not dx[0, 1, 3].isnan().any()


def sum_chain(B, N, H, others, D, half):
    """Additions on a weight gradient term's way in a lane: rows that a group of lanes carries in a tile, times the tiles that a
    workgroup walks (a row's lanes: a power of two from 4 on that holds its items of 16 elements; 256 threads; tokens of a tile: 4
    rows a thread, 2048 angles and two workgroups for each of 256 CUs; 768 workgroups for both sides)."""
    items = -(-half // 8) + -(-(D - 2 * half) // 16)
    lanes = next(n for n in (4, 8, 16, 32) if n >= items)
    tokens = max(1, min(4 * 256 // lanes // H, 2048 // half, B * N // 512, N))
    tiles = B * -(-N // tokens)
    groups = min(tiles, max(1, H * 768 // (H + others)))
    return -(-tiles // groups) * -(-tokens * H * lanes // 256), tokens


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('dtype, wdtype', [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                           (torch.float32, torch.bfloat16)], ids=str)
@pytest.mark.parametrize('shape', [(1, 1500, 2, 1, 64, 32), (3, 777, 4, 2, 48, 24), (2, 1201, 1, 3, 128, 64), (1, 4099, 5, 1, 80, 40),
                                   (2, 2500, 8, 2, 72, 12), (1, 6007, 1, 1, 36, 18), (64, 19, 12, 12, 64, 16), (1200, 1, 2, 1, 17, 8),
                                   (2, 700, 3, 2, 256, 128), (1, 3001, 2, 2, 255, 100)], ids=str)
def test_tiles_of_several_tokens_against_float64(shape, dtype, wdtype, layout):
    """From 1024 tokens on a tile has more than one: results and gradients of every leaf."""
    from streamvoxel_amd.stream.rotary import norm_rotary
    B, N, H, Hk, D, half = shape
    _case(f'norm_rotary tiles {shape} {dtype} {wdtype} {layout}')
    assert sum_chain(B, N, H, Hk, D, half)[1] > 1 or N == 1
    q, k, wq, wk, dq, dk = inputs(B, N, H, Hk, D, dtype, wdtype, D + N)
    g = torch.Generator().manual_seed(1)
    positions = torch.randint(-50, 200000, (B, N), generator=g)
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    amplitude, eps = 1.25, 1e-5
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    y = norm_rotary(*leaves, positions.to(DEV), freq.to(DEV), eps=eps, layout=layout, amplitude=amplitude)
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    for i, (x, w, dy) in enumerate(((q, wq, dq), (k, wk, dk))):
        ref = reference(x, w, positions, freq, layout, amplitude, eps, dy)
        check(y[i], ref['y'], 'y')
        check(grads[i], ref['dx'], 'dx')
        # (The bound that is there counts a term for every 8 rows; a lane's own additions here.)
        value, err = ref['dw']
        rows = B * x.shape[1] * N
        chain = sum_chain(B, N, x.shape[1], H + Hk - x.shape[1], D, half)[0]
        check(grads[2 + i], (value, err / (25 + 74 + rows / 8) * (25 + 74 + chain)), 'dw')
