"""CPU checks of what an append may change of a window's keys (PagedContext.tail)."""
import pytest
import torch

from streamvoxel_amd.stream.paged import PagedContext


@pytest.mark.parametrize('page, block', [(64, 64), (64, 16), (128, 32)])
def test_the_block_that_the_keys_end_inside_of(page, block, monkeypatch):
    monkeypatch.setattr(PagedContext, '_send', staticmethod(lambda to, values: to.copy_(torch.tensor(values, dtype=torch.int32))))
    ctx = PagedContext(2, 2, 3, 8, 9, 'cpu', page_size=page, kv_dtype='int8', block=block)
    ctx.resize(0, 5)
    for held in (0, 1, block - 1, block, block + 1, page - 1, page, page + 7, 2 * page + block, 2 * page + block + 3):
        ctx.resize(1, held)
        for pool in (ctx.k, ctx.v, ctx.k_exponents, ctx.v_exponents):
            for t in pool:
                t.copy_(torch.randint(0, 100, t.shape))
        parts = ctx.tail(1, 1)
        assert len(parts) == (0 if held % block == 0 else 4)
        was = [t.clone() for t in (ctx.k[1], ctx.v[1], ctx.k_exponents[1], ctx.v_exponents[1])]
        if not parts:
            continue
        first = held // block * block                         # the keys of the block, wherever its page lies
        number = int(ctx.table[1, first // page])
        rows, e = slice(first % page, first % page + held - first), first % page // block
        for t in (ctx.k[1], ctx.v[1]):
            t[number, :, rows] = -1
        for t in (ctx.k_exponents[1], ctx.v_exponents[1]):
            t[number, :, e] = 200
        for part, copy in parts:
            part.copy_(copy)
        assert all(torch.equal(a, b) for a, b in zip(was, (ctx.k[1], ctx.v[1], ctx.k_exponents[1], ctx.v_exponents[1])))
    for kind in ('bf16', 'fp8'):
        other = PagedContext(1, 1, 1, 8, 4, 'cpu', kv_dtype=kind)
        other.resize(0, 70)
        assert other.tail(0, 0) == []
