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
