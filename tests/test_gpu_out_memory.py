"""Where the results of rotary, norm_rotary, paged_append, paged_read and paged_attention may not go: refused before a launch."""
import pytest
import torch

from test_gpu_paged_int8 import Int8Pool, queries

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def sliding(B, H, n, D, dtype=torch.bfloat16):
    """[B, H, n, D] rows that slide by 8 elements."""
    return torch.zeros(B, H, 8 * (n - 1) + D, dtype=dtype, device=DEV).unfold(2, D, 8)


def test_rows_that_slide_over_each_other():
    from streamvoxel_amd.stream.paged import paged_append, paged_attention, paged_read
    from streamvoxel_amd.stream.rotary import norm_rotary, rotary
    x, k = [torch.randn(2, n, 5, 64, device=DEV).to(torch.bfloat16) for n in (4, 2)]
    p, f = torch.arange(5, device=DEV), torch.ones(32, dtype=torch.float64, device=DEV)
    bad = sliding(2, 4, 5, 64)
    assert bad.shape == x.shape and bad.stride(-1) == 1
    for out in (bad, bad.clone()):
        refused = out is bad
        for call in (lambda: rotary(x, p, f, out=out), lambda: rotary(out, p, f, out=out),
                     lambda: norm_rotary(x, k, None, None, p, f, out=(out, torch.empty_like(k))),
                     lambda: norm_rotary(k, x, None, None, p, f, out=(torch.empty_like(k), out)),
                     lambda: norm_rotary(out, k, None, None, p, f, out=(out, k))):
            if refused:
                with pytest.raises(ValueError, match='place for every element'):
                    call()
            else:
                call()
    pool = Int8Pool([100, 7], 2, 64, 64, 1, 32)
    args, e = pool.args(), pool.exponents()
    with pytest.raises(ValueError, match='place for every element'):
        paged_attention(queries(2, 4, 5, 64, 1), *args, out=bad, **e)
    for out in ((sliding(2, 2, 5, 64), torch.empty_like(k)), (torch.empty_like(k), sliding(2, 2, 5, 64))):
        with pytest.raises(ValueError, match='place for every element'):
            paged_read(*args, 5, out=out, **e)
    pages = sliding(4, 2, 16, 64)
    with pytest.raises(ValueError, match='place for every element'):
        paged_append(k, k, torch.empty_like(pages), pages, torch.zeros(2, 1, dtype=torch.int32, device=DEV),
                     torch.full((2,), 5, dtype=torch.int32, device=DEV))
