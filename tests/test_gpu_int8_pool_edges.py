"""An int8 paged cache on the GPU where a value, a scale or a failure is out of the ordinary: infinities beside good keys,
scores scaled by next to nothing or by far too much.

Tolerances. Append: what is compared is the append itself on inputs that differ in the elements under test alone: equal codes.
Attention: that of test_gpu_paged_int8.py."""
import math

import pytest
import torch

from test_gpu_paged import queries
from test_gpu_paged_int8 import Int8Pool, check

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def _case(msg):
    print(f'[gpu-case] {msg}', flush=True)


def fresh(pages, H, page, D, block):
    k, v = [torch.zeros(pages, H, page, D, dtype=torch.int8, device=DEV) for _ in 'kv']
    e = {name: torch.zeros(pages, H, page // block, dtype=torch.uint8, device=DEV) for name in ('k_exponents', 'v_exponents')}
    return k, v, e


@pytest.mark.parametrize('layout, half', [(None, 0), ('half', 24), ('half', 5), ('interleaved', 24), ('interleaved', 7)])
@pytest.mark.parametrize('D, block', [(48, 16), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize('older, n', [(0, 1), (20, 1), (3, 9), (0, 64), (40, 90), (5, 200)])
def test_an_infinity_or_nan_beside_good_keys(older, n, D, block, layout, half):
    """The other elements, older rows among them, are held as if a zero stood in its place: it is the largest number of its
    block (NaN 0), and sets `bad`."""
    from streamvoxel_amd.stream.paged import paged_append
    _case(f'infinities older={older} n={n} D={D} block={block} {layout} {half}')
    H, page = 3, 64
    g = torch.Generator().manual_seed(D + n)
    total = older + n
    pages = -(-total // page)
    table = torch.randperm(pages, generator=g).to(torch.int32)[None].to(DEV)
    rows = torch.randn(2, 1, H, total, D, generator=g).to(torch.bfloat16)
    how = {}
    if layout:
        how = dict(layout=layout, frequencies=(1.0 / (1.3 + torch.arange(half, dtype=torch.float64))).to(DEV))
    # (row, head, element, value): in the first, a middle and the last new row, in either half of a row.
    marks = [(older, 0, 1, math.inf), (older + n // 2, 1, D // 2 + 3, -math.inf), (total - 1, 2, 4, math.nan),
             (total - 1, 0, D - 2, math.inf)]
    if layout:                       # (what an infinity is turned to depends on the signs of cos and sin alone)
        pair = lambda d: (None if d >= 2 * half else (d % half, d % half + half) if layout == 'half' else (d & ~1, d | 1))
    else:
        pair = lambda d: None
    wild, calm = rows.clone(), rows.clone()
    for j, h, d, value in marks:
        for e in pair(d) or (d,):
            wild[:, 0, h, j, e] = calm[:, 0, h, j, e] = 0.0
    for j, h, d, value in marks:
        wild[:, 0, h, j, d] = value
    pools = []
    for x in (calm, wild):
        k, v, e = fresh(pages, H, page, D, block)
        if older:
            paged_append(*rows[:, :, :, :older].to(DEV), k, v, table, torch.tensor([older], dtype=torch.int32, device=DEV), **e, **how)
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        paged_append(*x[:, :, :, older:].to(DEV), k, v, table, torch.tensor([total], dtype=torch.int32, device=DEV), bad=bad, **e, **how)
        at = table[0].cpu().long()
        line = lambda t: t.cpu()[at].transpose(0, 1).reshape(H, -1, *t.shape[3:])
        pools.append((line(k), line(v), line(e['k_exponents']), line(e['v_exponents']), int(bad)))
    (ck, cv, cke, cve, calm_bad), (wk, wv, wke, wve, wild_bad) = pools
    assert calm_bad == 0 and wild_bad == 1
    assert torch.equal(cke, wke) and torch.equal(cve, wve)
    code = lambda x: 0 if math.isnan(x) else int(math.copysign(127, x))
    for j, h, d, value in marks:
        cv[h, j, d] = code(value)
        if layout and pair(d):
            a, b = pair(d)
            angle = j * float(how['frequencies'][d % half if layout == 'half' else d // 2])
            c, s = math.cos(angle), math.sin(angle)
            if d == a:
                turned = value * c, (math.nan if s == 0 else value * s)
            else:
                turned = (math.nan if s == 0 else -value * s), value * c
            ck[h, j, a], ck[h, j, b] = map(code, turned)
        else:
            ck[h, j, d] = code(value)
    assert torch.equal(ck, wk) and torch.equal(cv, wv)


@pytest.mark.parametrize('older', [0, 2])
@pytest.mark.parametrize('n', [1, 40, 62])
@pytest.mark.parametrize('D', [48, 128])
def test_infinities_among_zeros(n, older, D):
    """A block that has nothing else but zeros holds an infinity as the largest number there is; a finite value anywhere in it,
    or a key in front, sets the block's scale in its place."""
    from streamvoxel_amd.stream.paged import paged_append
    H, page, block = 2, 64, 64
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    length = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)
    for others in (0.0, 3.0):
        k, v, e = fresh(1, H, page, D, block)
        old = torch.full((1, H, older, D), 0.75, dtype=torch.bfloat16, device=DEV)
        if older:
            paged_append(old, old, k, v, table, length(older), **e)
        x = torch.zeros(1, H, n, D, dtype=torch.bfloat16)
        x[0, 1, n // 2, 5], x[0, 0, n - 1, 6] = -math.inf, math.inf
        if others:
            x[0, :, 0, 7] = others
        x, bad = x.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        paged_append(x, x, k, v, table, length(older + n), bad=bad, **e)
        exponent = 122 if others else (120 if older else 248)      # 3 = 96 * 2^-5, 0.75 = 96 * 2^-7
        want = torch.zeros(H, page, D, dtype=torch.int8)
        want[:, :older] = 24 if others else 96
        want[1, older + n // 2, 5], want[0, older + n - 1, 6] = -127, 127
        if others:
            want[:, older, 7] = 96
        assert int(bad) == 1 and torch.equal(k[0].cpu(), want) and torch.equal(v, k)
        assert (e['k_exponents'] == exponent).all() and (e['v_exponents'] == exponent).all()


@pytest.mark.parametrize('n', [1, 3, 40, 200])
@pytest.mark.parametrize('scale', [1e-2, 1e-8, 1e-25, 1e-38, 1e-42], ids=str)
@pytest.mark.parametrize('D, H, heads, page, block', [(64, 4, 2, 64, 64), (48, 3, 3, 16, 16), (128, 8, 1, 128, 32)])
def test_scores_scaled_by_next_to_nothing(D, H, heads, page, block, scale, n):
    """Blocks of zeros (their power of two is 2^-126), blocks that end inside and keys masked in them: the weights are all but
    equal, and keys that a token does not see stay out."""
    from streamvoxel_amd.stream.paged import paged_attention
    _case(f'int8 scale={scale} n={n} D={D} page={page} block={block}')
    pool = Int8Pool([70, 0, 333, 1, 1000], heads, D, page, 5, block)
    for at in (0, pool.k.shape[0] // 2):                       # every second page: codes of zero under the least exponent
        pool.k[at::2] = 0
        pool.ke[at::2] = 1
    q = queries(5, H, n, D, n)
    for how in (dict(causal=True), dict(causal=False), dict(causal=True, window=20, sinks=3)):
        got = paged_attention(q, *pool.args(), scale=scale, **how, **pool.exponents())
        check(got, q, pool, scale=scale, **how)


@pytest.mark.parametrize('n', [1, 40])
def test_queries_of_zeros_at_the_largest_scales(n):
    """Scores of 0 times whatever is still 0: every key in sight weighs the same."""
    from streamvoxel_amd.stream.paged import paged_attention
    pool = Int8Pool([70, 333], 2, 64, 64, 5, 32)
    pool.ke[:] = 248
    q = torch.zeros(2, 4, n, 64, dtype=torch.bfloat16, device=DEV)
    for scale in (1.0, 200.0, 1e30):
        got = paged_attention(q, *pool.args(), scale=scale, causal=True, **pool.exponents())
        check(got, q, pool, scale=scale)


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'int8'])
@pytest.mark.parametrize('n', [1, 3, 100])
def test_a_window_over_everything_has_the_bits_of_none(n, kind):
    from streamvoxel_amd.stream.paged import paged_attention
    from test_gpu_paged_int8 import pool_of
    pool = pool_of(kind, [3000, 300, 500], 2, 64, 64, 3)
    q = queries(3, 4, n, 64, n)
    want = paged_attention(q, *pool.args(), causal=True, **pool.exponents())
    for window, sinks in ((3000, 0), (1 << 40, 0), (1 << 62, 1 << 62)):
        assert torch.equal(paged_attention(q, *pool.args(), causal=True, window=window, sinks=sinks, **pool.exponents()), want)
