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


def test_memory_that_the_call_reads():
    """One buffer holds a result's rows and, inside of them, what a call reads beside its rows."""
    from streamvoxel_amd.stream.paged import paged_attention, paged_read
    from streamvoxel_amd.stream.rotary import norm_rotary, rotary
    B, H, n, D = 2, 4, 8, 64

    def inside(t):
        """A [B, H, n, D] result whose buffer begins with what t holds, and t there."""
        buffer = torch.zeros(B * H * n * D, dtype=torch.bfloat16, device=DEV)
        there = buffer.view(torch.uint8)[:t.nbytes].view(t.dtype).view(t.shape)
        there.copy_(t)
        return buffer.view(B, H, n, D), there

    x = torch.randn(B, H, n, D, device=DEV).to(torch.bfloat16)
    p, f = torch.arange(n, device=DEV), torch.ones(32, dtype=torch.float64, device=DEV)
    w = torch.ones(D, device=DEV)
    for which, t in enumerate((p, f, w, w)):
        out, there = inside(t)
        args = [p, f, w, w]
        args[which] = there
        for pair in ((out, torch.empty_like(x)), (torch.empty_like(x), out)):
            with pytest.raises(ValueError, match='share memory'):
                norm_rotary(x, x, args[2], args[3], args[0], args[1], out=pair)
        if which < 2:
            with pytest.raises(ValueError, match='share memory'):
                rotary(x, args[0], args[1], out=out)
    pool = Int8Pool([100, 7], H, D, 64, 1, 32)
    k, v, table, L = pool.args()
    e = pool.exponents()
    cu, bad = torch.tensor([0, 8, 16], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    names = ('page_table', 'lengths', 'k_exponents', 'v_exponents', 'bad')
    held = dict(page_table=table, lengths=L, bad=bad, **e)
    for name in names:
        out, there = inside(held[name])
        how = {**held, name: there}
        with pytest.raises(ValueError, match='share memory'):
            paged_attention(x, k, v, out=out, **how)
        for pair in ((out, torch.empty_like(out)), (torch.empty_like(out), out)):
            with pytest.raises(ValueError, match='share memory'):
                paged_read(k, v, n=n, out=pair, **how)
    out, there = inside(cu)
    packed = out.view(H, B * n, D)
    with pytest.raises(ValueError, match='share memory'):
        paged_attention(x.view(H, B * n, D), k, v, out=packed, cu_queries=there, **held)
    with pytest.raises(ValueError, match='share memory'):
        paged_read(k, v, n=B * n, out=(packed, torch.empty_like(packed)), cu_keys=there, **held)
    pages = torch.zeros(4, H, 64, D, dtype=torch.bfloat16, device=DEV)
    for kv in ((pages, torch.zeros_like(pages)), (torch.zeros_like(pages), pages)):
        with pytest.raises(ValueError, match='share memory'):
            paged_attention(x, *kv, table, L, out=pages.view(-1)[:x.numel()].view(x.shape))


def test_queries_and_keys_that_are_one_tensor():
    """Their results may be fresh or lie elsewhere, but not in the tensor that the other side still reads."""
    from streamvoxel_amd.stream.rotary import norm_rotary
    x = torch.randn(2, 4, 8, 64, device=DEV).to(torch.bfloat16)
    p, f = torch.arange(8, device=DEV), torch.ones(32, dtype=torch.float64, device=DEV)
    w, v = torch.rand(64, device=DEV), torch.rand(64, device=DEV)
    want = norm_rotary(x, x, w, v, p, f)
    other, again = torch.empty_like(x), x.view(2, 4, 8, 64)
    for q, k, out in ((x, x, (x, x)), (x, x, (x, other)), (x, x, (other, x)), (x, again, (x, again)), (x, again, (x, other)),
                      (x, again, (other, again)), (x, x, (other, other)), (x, x[:, 1:3], (x, other[:, :2])),
                      (x[:, 1:3], x, (other[:, :2], x))):
        with pytest.raises(ValueError, match='memory'):
            norm_rotary(q, k, w, v, p, f, out=out)
    got = norm_rotary(x, x, w, v, p, f, out=(other, torch.empty_like(x)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    rows = torch.randn(2, 8, 6, 64, device=DEV).to(torch.bfloat16)
    q, k = rows[:, :, :4].transpose(1, 2), rows[:, :, 4:].transpose(1, 2)
    want = norm_rotary(q, k, w, v, p, f)
    spare = torch.empty_like(rows)
    for out in ((spare[:, :, :4].transpose(1, 2), k), (q, spare[:, :, 4:].transpose(1, 2)), (q, k)):
        keep = rows.clone()
        got = norm_rotary(q, k, w, v, p, f, out=out)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        rows.copy_(keep)
    alone = norm_rotary(q, None, w, None, p, f, out=(q, None))
    assert alone[0] is q and torch.equal(q, want[0])
