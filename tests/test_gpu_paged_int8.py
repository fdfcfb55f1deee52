"""An int8 paged cache on the GPU: the append that holds keys in blocks, the reading back (of every kind of pool), the attention
over it, and attention through a sliding window over every kind of pool; against plain float64 on the host.

Tolerances. Append: a block's exponent is exact unless its largest magnitude lies within 16 * 2^-24 of the border (a rotated
value is off by 8 * 2^-24 of |x_a| + |x_b|, test_gpu_rotary.py); a code is off by half a step, and that error; where nothing
turns, codes and exponents are exact, and so are the older ones of a block. Reading back is exact. Attention: as
test_gpu_paged.py, whose arithmetic holds for any storage that decodes to bf16 exactly, and for any set of keys that a row
sees."""
import math

import pytest
import torch

from test_gpu_paged import Pool, queries

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
E = 2.0 ** -24


def _case(msg):
    print(f'[gpu-case] {msg}', flush=True)


class Int8Pool(Pool):
    """A pool of codes with an exponent for every `block` keys; random ones where no window's keys lie, exponents up to 255
    among them."""

    def __init__(self, lengths, heads, D, page, seed, block, **how):
        super().__init__(lengths, heads, D, page, seed, 'bf16', clean=True, **how)
        g = torch.Generator().manual_seed(seed + 1)
        self.block = block
        shape = (self.pages, heads, page // block)
        self.ke, self.ve = [torch.randint(119, 123, shape, generator=g).to(torch.uint8) for _ in 'kv']
        used = torch.zeros(self.pages, page // block, dtype=torch.bool)
        for b, L in enumerate(lengths):
            for j in range(-(-max(L, 0) // page)):
                used[self.table[b, j], :-(-min(page, L - j * page) // block)] = True
        for e in (self.ke, self.ve):
            e[~used[:, None].expand(-1, heads, -1)] = 255
        self.k, self.v = [(t.float() * 48).round().clamp(-127, 127).to(torch.int8) for t in (self.k, self.v)]

    def exponents(self):
        return dict(k_exponents=self.ke.to(DEV), v_exponents=self.ve.to(DEV))

    def rows(self, b):
        L = max(self.lengths[b], 0)
        page = self.table[b, :-(-L // self.page)].long()
        out = []
        for t, e in ((self.k, self.ke), (self.v, self.ve)):
            x = t[page].double() * 2.0 ** (e[page].double() - 127).repeat_interleave(self.block, -1)[..., None]
            out.append(x.transpose(0, 1).reshape(self.heads, -1, self.D)[:, :L])
        return out


def pool_of(kind, lengths, heads, D, page, seed, block=16, **how):
    if kind == 'int8':
        how.pop('clean', None)
        return Int8Pool(lengths, heads, D, page, seed, min(block, page), **how)
    return Pool(lengths, heads, D, page, seed, kind, **how)


def attend64(q, k, v, seen, scale):
    """(out, allowed error) of one window: q [H, n, D], k, v [heads, L, D] float64, seen [n, L]."""
    H, n, D = q.shape
    L, G = k.shape[1], H // k.shape[0]
    if L == 0 or n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    # (What no row sees may be NaN or infinite.)
    k = torch.where(seen.any(0)[None, :, None], k, torch.zeros_like(k))
    v = torch.where(seen.any(0)[None, :, None], v, torch.zeros_like(v))
    s = scale * q @ k.transpose(1, 2)
    off = 2.0 ** -24 * (D * scale * (q.abs() @ k.abs().transpose(1, 2)) + 4 * (1 + s.abs()))
    s, off = s.masked_fill(~seen, -math.inf), off.masked_fill(~seen, 0.0)
    w = (s - s.amax(-1, keepdim=True).clamp(min=-1e300)).exp()
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total.clamp(min=1e-300), torch.zeros_like(w))
    out, A = w @ v, w @ v.abs()
    err = (2 * 2.0 ** -8 + 2 * off.amax(-1, keepdim=True)) * A
    return out, err + 2.0 ** -8 * (out.abs() + err)


def visible(L, n, causal, window, sinks, held=None):
    """[n, L] of the keys that each token sees; `held`: the length that the tokens count from, where it is another."""
    j, p = torch.arange(L)[None], (L if held is None else held) - n + torch.arange(n)[:, None]
    if not causal:
        return torch.ones(n, L, dtype=torch.bool)
    if window is None:
        return j <= p
    return (j <= p) & ((j > p - window) | (j < sinks))


def check(got, q, pool, causal=True, window=None, sinks=0, cu=None, scale=None):
    scale = 1 / math.sqrt(pool.D) if scale is None else scale
    got, q = got.cpu().double(), q.cpu().double()
    for b in range(len(pool.lengths)):
        cut = (lambda t: t[b]) if cu is None else (lambda t: t[:, cu[b]:cu[b + 1]])
        k, v = pool.rows(b)
        out, err = attend64(cut(q), k, v, visible(k.shape[1], cut(q).shape[1], causal, window, sinks, pool.lengths[b]), scale)
        off = (cut(got) - out).abs()
        assert not torch.isnan(off).any(), b
        assert (off <= err).all(), (b, (off - err).max().item(), off.max().item())


LENGTHS = [[0, 1, 15, 16, 17], [63, 64, 65, 31, 33], [500, 129, 0, 700, 128], [3001], [1537, 40, 9000]]


@pytest.mark.parametrize('block', [16, 32, 64])
@pytest.mark.parametrize('lengths', LENGTHS, ids=lambda x: '-'.join(map(str, x)))
@pytest.mark.parametrize('n, causal', [(1, False), (1, True), (2, True), (7, False), (40, True), (130, True), (130, False)])
@pytest.mark.parametrize('D, H, heads, page', [(64, 4, 4, 64), (48, 6, 2, 64), (128, 8, 1, 128), (96, 3, 3, 128), (8, 2, 1, 1024),
                                               (72, 4, 2, 64)])
def test_int8_attention_against_float64(lengths, n, causal, D, H, heads, page, block):
    from streamvoxel_amd.stream.paged import paged_attention
    _case(f'int8 attention {lengths} n={n} causal={causal} D={D} H={H}/{heads} page={page} block={block}')
    pool = Int8Pool(lengths, heads, D, page, sum(lengths) + n, block)
    q = queries(len(lengths), H, n, D, n + D)
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = paged_attention(q, *pool.args(), causal=causal, bad=bad, **pool.exponents())
    assert int(bad) == 0
    check(got, q, pool, causal)


@pytest.mark.parametrize('page, block', [(16, 16), (32, 16), (32, 32)])
@pytest.mark.parametrize('n', [1, 60])
def test_int8_small_pages(n, page, block):
    from streamvoxel_amd.stream.paged import paged_attention
    pool = Int8Pool([700, 3, 96, 41], 2, 64, page, n, block, token_major=True)
    q = queries(4, 4, n, 64, n)
    check(paged_attention(q, *pool.args(), causal=True, **pool.exponents()), q, pool)


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'int8'])
@pytest.mark.parametrize('D', range(8, 129, 8))
def test_every_head_width(D, kind):
    from streamvoxel_amd.stream.paged import paged_attention
    for n, page in ((1, 16), (1, 64), (50, 16), (50, 64)):
        pool = pool_of(kind, [333, 64, 5], 2, D, page, D + n, block=32)
        q = queries(3, 4, n, D, D)
        for how in (dict(window=70, sinks=3), dict(window=None)):
            check(paged_attention(q, *pool.args(), causal=True, **how, **pool.exponents()), q, pool, **how)


WINDOWS = [(1, 0), (1, 1), (5, 4), (64, 0), (65, 5), (128, 130), (300, 16), (1000, 1), (17, 100000)]


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'int8'])
@pytest.mark.parametrize('window, sinks', WINDOWS, ids=str)
@pytest.mark.parametrize('lengths', LENGTHS, ids=lambda x: '-'.join(map(str, x)))
@pytest.mark.parametrize('n', [1, 3, 40, 300])
@pytest.mark.parametrize('D, H, heads, page', [(64, 4, 4, 64), (128, 8, 1, 32), (40, 6, 2, 16)])
def test_window_attention_against_float64(lengths, n, window, sinks, D, H, heads, page, kind):
    """NaN (int8: exponents of 255) in every row that holds no key."""
    from streamvoxel_amd.stream.paged import paged_attention
    _case(f'window attention {lengths} n={n} window={window} sinks={sinks} D={D} H={H}/{heads} page={page} {kind}')
    pool = pool_of(kind, lengths, heads, D, page, sum(lengths) + n)
    q = queries(len(lengths), H, n, D, n + D)
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = paged_attention(q, *pool.args(), causal=True, window=window, sinks=sinks, bad=bad, **pool.exponents())
    assert int(bad) == 0
    check(got, q, pool, window=window, sinks=sinks)


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'int8'])
@pytest.mark.parametrize('window, sinks', [(40, 3), (700, 100)])
@pytest.mark.parametrize('counts', [[1, 0, 5, 1, 1, 200, 33], [0, 0, 3], [1, 1, 1, 1], [129, 1], [600, 1]], ids=str)
@pytest.mark.parametrize('D, H, heads, page', [(64, 4, 1, 16), (128, 4, 4, 64), (96, 8, 2, 32)])
def test_packed_windows(counts, D, H, heads, page, window, sinks, kind):
    """Tiles beside single tokens; rows in front of the first border and behind the last stay as they were."""
    from streamvoxel_amd.stream.paged import paged_attention
    g = torch.Generator().manual_seed(len(counts))
    lengths = [n + int(torch.randint(0, 3000, (1,), generator=g)) for n in counts]
    pool = pool_of(kind, lengths, heads, D, page, sum(lengths))
    cu = [3]
    for n in counts:
        cu.append(cu[-1] + n)
    T = cu[-1] + 5
    q = queries(1, H, T, D, T)[0]
    out = torch.full_like(q, 7.0)
    borders = torch.tensor(cu, dtype=torch.int32, device=DEV)
    for how in (dict(window=window, sinks=sinks), dict(window=None)):
        got = paged_attention(q, *pool.args(), cu_queries=borders, causal=True, out=out, **how, **pool.exponents())
        check(got, q, pool, cu=cu, **how)
        assert (got[:, :3] == 7).all() and (got[:, cu[-1]:] == 7).all()


@pytest.mark.parametrize('kind', ['bf16', 'fp8'])
@pytest.mark.parametrize('D, heads, page', [(64, 1, 64), (128, 2, 16)])
@pytest.mark.parametrize('n', [1, 2, 40, 200])
@pytest.mark.parametrize('window, sinks', [(33, 5), (200, 0), (1, 70)])
def test_what_a_token_does_not_see_does_not_reach_it(window, sinks, n, D, heads, page, kind):
    """NaN and infinite keys and values in front of the windows, behind the first keys, and where some tokens of a tile see
    them and others do not: the ones that see them are not finite, the others as without."""
    from streamvoxel_amd.stream.paged import paged_attention
    L = 900
    pool = Pool([L], heads, D, page, n + window, kind)
    q = queries(1, 2 * heads, n, D, n)
    k, v = pool.rows(0)
    want, err = attend64(q[0].cpu().double(), k, v, visible(L, n, True, window, sinks), D ** -0.5)
    codes = dict(bf16=[math.nan, math.inf, -math.inf], fp8=[math.nan] * 3)[kind]
    spots = [sinks, max(sinks, L - n - window), max(sinks, L - n - window + n // 2), L - 1]
    seen = visible(L, n, True, window, sinks)
    for i, j in enumerate(spots):
        for pages in (pool.k, pool.v):
            held = pages[pool.table[0, j // page], :, j % page].clone()
            value = torch.full((heads, D), codes[i % 3]).to(pages.dtype)
            if pages is pool.k:
                value[:, 1:] = held[:, 1:]
            pages[pool.table[0, j // page], :, j % page] = value
            got = paged_attention(q, *pool.args(), causal=True, window=window, sinks=sinks, **pool.exponents())
            sees = seen[:, j]
            same = got[0].cpu().double()[:, ~sees]
            assert same.isfinite().all(), (j, 'reached')
            assert ((same - want[:, ~sees]).abs() <= err[:, ~sees]).all(), j
            if pages is pool.v:
                assert not got[0][:, sees.to(DEV)].isfinite().any(), j
            pages[pool.table[0, j // page], :, j % page] = held


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'int8'])
@pytest.mark.parametrize('B, n, packed', [(90, 1, False), (200, 30, False), (1100, 1, True), (70, 9, True)])
def test_many_windows(B, n, packed, kind):
    from streamvoxel_amd.stream.paged import paged_attention
    _case(f'many windows B={B} n={n} packed={packed} {kind}')
    g = torch.Generator().manual_seed(B)
    counts = [int(c) for c in torch.randint(0, 2 * n + 1, (B,), generator=g)] if packed else [n] * B
    lengths = [c + int(x) for c, x in zip(counts, torch.randint(0, 400, (B,), generator=g))]
    lengths[B // 2] = 5000
    pool = pool_of(kind, lengths, 2, 64, 32, B)
    cu = None
    if packed:
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
    q = queries(1, 4, cu[-1], 64, B)[0] if packed else queries(B, 4, n, 64, B)
    borders = torch.tensor(cu, dtype=torch.int32, device=DEV) if packed else None
    for how in (dict(window=100, sinks=4), dict(window=2000, sinks=0), dict(window=None)):
        got = paged_attention(q, *pool.args(), cu_queries=borders, causal=True, **how, **pool.exponents())
        check(got, q, pool, cu=cu, **how)


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'int8'])
@pytest.mark.parametrize('n', [1, 70])
def test_bad_pages_and_lengths(n, kind):
    """A bad page reads as zeros, a length past the table's row is cut, though the window slides from the whole length; both
    set the flag. A negative length is empty."""
    from streamvoxel_amd.stream.paged import paged_attention
    pool = pool_of(kind, [640, 300], 2, 64, 64, n, block=64, clean=True)
    q = queries(2, 4, n, 64, n)
    args = list(pool.args())
    for page, at in ((-1, 9), (pool.pages, 9), (1 << 30, 0)):
        table = pool.table.clone()
        table[0, at] = page
        args[2] = table.to(DEV)
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = paged_attention(q, *args, causal=True, window=100, sinks=5, bad=bad, **pool.exponents())
        assert int(bad) == 1
        keep = pool.rows
        def rows(b):
            k, v = [t.clone() for t in keep(b)]
            if b == 0:
                k[:, 64 * at:64 * at + 64] = 0
                v[:, 64 * at:64 * at + 64] = 0
            return k, v
        pool.rows = rows
        check(got, q, pool, window=100, sinks=5)
        pool.rows = keep
    args[2] = pool.table[:, :8].contiguous().to(DEV)        # 512 of the 640 keys
    for window, sinks in ((200, 3), (200, 0), (50, 0), (50, 2), (600, 0)):
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = paged_attention(q, *args, causal=True, window=window, sinks=sinks, bad=bad, **pool.exponents())
        assert int(bad) == 1
        keep = pool.rows
        pool.rows = lambda b: [t[:, :512] for t in keep(b)]
        check(got, q, pool, window=window, sinks=sinks)
        pool.rows = keep
    args[2], args[3] = pool.table.to(DEV), torch.tensor([-5, 0], dtype=torch.int32, device=DEV)
    assert not paged_attention(q, *args, causal=True, window=50, sinks=2, **pool.exponents()).any()


def test_queries_that_overlap():
    """Queries as windows that slide over one sequence, 8 elements a token: their copies' results."""
    from streamvoxel_amd.stream.paged import paged_attention
    _case('overlapping queries')
    pool = pool_of('int8', [40, 17], 2, 64, 32, 3)
    query = torch.randn(2, 4, 8 * 6 + 64, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(DEV).unfold(2, 64, 8)
    got, want = (paged_attention(q, *pool.args(), causal=True, window=9, sinks=2, **pool.exponents())
                 for q in (query, query.contiguous()))
    assert torch.equal(got, want)
    check(got, query, pool, window=9, sinks=2)


def test_a_window_as_long_as_everything_is_no_window():
    """The same bits where every key is in sight and the kernels cut alike."""
    from streamvoxel_amd.stream.paged import paged_attention
    for kind in ('bf16', 'fp8', 'int8'):
        pool = pool_of(kind, [3000, 77, 500], 2, 64, 64, 3)
        for n in (1, 100):
            q = queries(3, 4, n, 64, n)
            want = paged_attention(q, *pool.args(), causal=True, **pool.exponents())
            for window, sinks in ((3000, 0), (1 << 40, 0), (1 << 62, 1 << 62)):
                got = paged_attention(q, *pool.args(), causal=True, window=window, sinks=sinks, **pool.exponents())
                check(got, q, pool)
                assert (got - want).abs().max() <= 2.0 ** -6


# ------------------------------------------------------------------------------------------------------ append and read

def hold64(rows, older, exponent, new, block):
    """Codes and exponent of one block of one head: `older` rows' codes [o, D] under `exponent`, new rows [m, D] float64."""
    most = new.abs().max().item() if new.numel() else 0.0
    e = 1
    if most > 0:
        mantissa, power = math.frexp(most)                   # 127 = 0.9921875 * 2^7
        e = (power - 7 if mantissa <= 0.9921875 else power - 6) + 127
    e = min(max(e, 1), 248)
    near = most > 0 and abs(math.log2(most / 127) - round(math.log2(most / 127))) < 16 * E / math.log(2)
    if older:
        e = max(e, min(exponent, 248))
        rows = torch.where(torch.tensor(exponent < e), (rows.double() * 2.0 ** (exponent - e)).round(), rows.double())
    codes = (new * 2.0 ** (127 - e)).round().clamp(-127, 127)
    return e, rows, codes, near


def turned64(key, where, freq, layout):
    if layout is None:
        return key, torch.zeros_like(key)
    half = len(freq)
    angle = where.double()[:, None] * freq
    c, s = angle.cos(), angle.sin()
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == 'half' else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    out, off = key.clone(), torch.zeros_like(key)
    out[..., a], out[..., b] = key[..., a] * c - key[..., b] * s, key[..., b] * c + key[..., a] * s
    off[..., a] = off[..., b] = 8 * E * (key[..., a].abs() + key[..., b].abs())
    return out, off


@pytest.mark.parametrize('layout, part', [(None, 0), ('half', 1.0), ('half', 0.6), ('interleaved', 1.0), ('interleaved', 0.3)])
@pytest.mark.parametrize('D, H, page, block', [(64, 4, 64, 64), (48, 3, 16, 16), (128, 1, 256, 64), (8, 2, 32, 16), (104, 5, 64, 32),
                                               (128, 17, 32, 32)])
@pytest.mark.parametrize('counts, packed, before', [([1, 1, 1], False, 0), ([40, 40, 40], False, 7), ([3, 0, 70, 1], True, 0),
                                                    ([200, 200], False, 0), ([1, 64, 16, 333, 1, 1], True, 0)])
def test_append_against_float64(counts, packed, before, D, H, page, block, layout, part):
    from streamvoxel_amd.stream.paged import paged_append
    _case(f'int8 append {counts} packed={packed} before={before} D={D} H={H} page={page} block={block} {layout} {part}')
    g = torch.Generator().manual_seed(sum(counts) + D)
    lengths = [n + before + int(x) for n, x in zip(counts, torch.randint(0, 150, (len(counts),), generator=g))]
    pool = Int8Pool(lengths, H, D, page, D, block)
    pool.ke[pool.ke < 255] -= 3                       # some blocks grow, some do not
    T = sum(counts) + (9 if packed else 0)
    spread = 2.0 ** torch.randint(-3, 4, (T, 1, 1), generator=g)
    key, value = [(torch.randn(T, H, D, generator=g) * spread).to(torch.bfloat16) for _ in 'kv']
    cu = None
    if packed:
        cu = [4]
        for n in counts:
            cu.append(cu[-1] + n)
    n = counts[0]
    shaped = lambda t: t.to(DEV).transpose(0, 1) if packed else t.to(DEV).view(len(counts), n, H, D).transpose(1, 2)
    freq = None
    if layout:
        half = max(1, int(part * D / 2))
        freq = 100.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    k, v, table, L = pool.args()
    e = pool.exponents()
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    paged_append(shaped(key), shaped(value), k, v, table, L, before=before, bad=bad, **e,
                 cu_tokens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV),
                 frequencies=None if freq is None else freq.to(DEV), layout=layout or 'half')
    assert int(bad) == 0
    got = {'k': (k.cpu(), e['k_exponents'].cpu()), 'v': (v.cpu(), e['v_exponents'].cpu())}
    want = {'k': (pool.k.clone(), pool.ke.clone()), 'v': (pool.v.clone(), pool.ve.clone())}
    first = cu[0] if packed else 0
    for b, n in enumerate(counts):
        at = torch.arange(n) + lengths[b] - before - n
        rows = slice(first, first + n)
        first += n
        turned, off = turned64(key[rows].double().transpose(0, 1), at, freq, layout)
        for side, new, off in (('k', turned, off), ('v', value[rows].double().transpose(0, 1), torch.zeros(H, n, D))):
            codes, exponents = want[side]
            for blk in sorted(set((at // block).tolist())):
                here = (at // block == blk).nonzero()[:, 0]
                j0 = int(at[here[0]])
                page_, row, older = int(pool.table[b, j0 // page]), j0 % page, j0 % block
                for h in range(H):
                    old = codes[page_, h, row - older:row]
                    eb, old, fresh, near = hold64(old, older, int(exponents[page_, h, row // block]), new[h, here], block)
                    ge = int(got[side][1][page_, h, row // block])
                    if ge != eb:
                        assert near and side == 'k' and layout, (b, h, blk, ge, eb)
                    step = 2.0 ** (ge - 127)
                    mine = got[side][0][page_, h, row:row + len(here)].double()
                    assert ((mine * step - new[h, here]).abs() <= step / 2 + off[h, here]).all(), (b, h, blk)
                    if ge == eb:
                        if not layout or side == 'v':
                            assert torch.equal(mine, fresh), (b, h, blk)
                        assert torch.equal(got[side][0][page_, h, row - older:row].double(), old.double()), (b, h, blk)
                    codes[page_, h, row - older:row + len(here)] = got[side][0][page_, h, row - older:row + len(here)]
                    exponents[page_, h, row // block] = ge
    for side in 'kv':                                 # everything else is as it was
        assert torch.equal(got[side][0], want[side][0]) and torch.equal(got[side][1], want[side][1])


@pytest.mark.parametrize('D', [48, 96])
def test_axial_append_has_the_bits_of_the_axial_rotation(D):
    from streamvoxel_amd.stream.paged import paged_append
    from streamvoxel_amd.stream.producer import axial_rope
    g = torch.Generator().manual_seed(D)
    n, H, page, block = 150, 3, 64, 32
    key = torch.randn(1, n, H, D, generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2)
    positions = (torch.rand(1, n, 3, generator=g) * 64 - 8).to(DEV)
    freq = (10000.0 ** (-torch.arange(0, D // 3, 2).float() / (D // 3))).to(DEV)
    pages = -(-n // page)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    L = torch.tensor([n], dtype=torch.int32, device=DEV)
    pools = []
    for x, how in ((axial_rope(key, positions, freq), {}), (key, dict(positions=positions, frequencies=freq, layout='axial'))):
        k, v = [torch.zeros(pages, H, page, D, dtype=torch.int8, device=DEV) for _ in 'kv']
        ke, ve = [torch.zeros(pages, H, page // block, dtype=torch.uint8, device=DEV) for _ in 'kv']
        paged_append(x, x, k, v, table, L, k_exponents=ke, v_exponents=ve, **how)
        pools.append((k, ke))
    assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1])


@pytest.mark.parametrize('block', [16, 64])
def test_a_block_filled_key_by_key(block):
    """Ascending magnitudes, which make the block grow with all but every key: what stands there at the end is off by less
    than a step of the last scale, and by half of one where the block was written at once."""
    from streamvoxel_amd.stream.paged import paged_append, paged_read
    D, H, n = 64, 2, 64
    g = torch.Generator().manual_seed(block)
    x = (torch.randn(1, H, n, D, generator=g) * (1.13 ** torch.arange(n))[:, None]).to(torch.bfloat16)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    for step in (1, 3, n):
        k, v = [torch.full((1, H, 64, D), 77, dtype=torch.int8, device=DEV) for _ in 'kv']
        ke, ve = [torch.full((1, H, 64 // block), 255, dtype=torch.uint8, device=DEV) for _ in 'kv']
        for at in range(0, n, step):
            m = min(step, n - at)
            L = torch.tensor([at + m], dtype=torch.int32, device=DEV)
            part = x[:, :, at:at + m].to(DEV)
            paged_append(part, part, k, v, table, L, k_exponents=ke, v_exponents=ve)
        got = paged_read(k, v, table, L, n, k_exponents=ke, v_exponents=ve)
        scale = 2.0 ** (ke.cpu().double() - 127).repeat_interleave(block, -1)[..., None]
        off = (got[0].cpu().double() - x.double()).abs() / scale
        assert off.max() <= (0.5 if step == n else 1.0)
        assert torch.equal(got[0], got[1])
        most = x.double().abs().amax(-1).unflatten(-1, (-1, block)).amax(-1)
        assert torch.equal(ke[:, :, :].cpu().double() - 127, torch.ceil(torch.log2(most / 127)))


def test_what_int8_cannot_hold():
    """Infinities as the largest number, NaN as 0, both flagged; zeros; the largest and the smallest values."""
    from streamvoxel_amd.stream.paged import paged_append, paged_read
    D, H = 8, 1
    table = torch.tensor([[0]], dtype=torch.int32, device=DEV)
    L = torch.tensor([16], dtype=torch.int32, device=DEV)
    for fill, flagged, want in ((math.inf, 1, 127 * 2.0 ** 121), (-math.inf, 1, -127 * 2.0 ** 121), (math.nan, 1, 0.0), (0.0, 0, 0.0),
                                (3.3895e38, 0, 127 * 2.0 ** 121), (2.0 ** -126, 0, 2.0 ** -126), (2.0 ** -130, 0, 0.0)):
        x = torch.zeros(1, H, 16, D)
        x[0, 0, 3, 2] = fill
        x = x.to(torch.bfloat16).to(DEV)
        k, v = [torch.zeros(1, H, 16, D, dtype=torch.int8, device=DEV) for _ in 'kv']
        ke, ve = [torch.zeros(1, H, 1, dtype=torch.uint8, device=DEV) for _ in 'kv']
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        paged_append(x, x, k, v, table, L, k_exponents=ke, v_exponents=ve, bad=bad)
        assert int(bad) == flagged, fill
        got = paged_read(k, v, table, L, 16, k_exponents=ke, v_exponents=ve)[0]
        assert float(got[0, 0, 3, 2]) == want, (fill, float(got[0, 0, 3, 2]))
        assert got.abs().sum() == abs(want) and 1 <= int(ke.item()) <= 248


def test_append_outside_the_table_or_the_pool_writes_nothing():
    from streamvoxel_amd.stream.paged import paged_append
    H, D, page = 2, 64, 16
    x = torch.ones(1, H, 40, D, dtype=torch.bfloat16, device=DEV)
    for table, length, first in (([[0, 5, 1]], 40, None), ([[0, -1, 1]], 40, None), ([[0, 1]], 40, None), ([[0, 1, 2]], 30, None)):
        k, v = [torch.full((3, H, page, D), 9, dtype=torch.int8, device=DEV) for _ in 'kv']
        ke, ve = [torch.full((3, H, 1), 100, dtype=torch.uint8, device=DEV) for _ in 'kv']
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        paged_append(x, x, k, v, torch.tensor(table, dtype=torch.int32, device=DEV),
                     torch.tensor([length], dtype=torch.int32, device=DEV), k_exponents=ke, v_exponents=ve, bad=bad)
        assert int(bad) == 1
        where = torch.arange(40) + length - 40
        want = torch.full((3, page), 9)
        for j in where.tolist():
            if 0 <= j < 16 * len(table[0]) and 0 <= table[0][j // 16] < 3:
                want[table[0][j // 16], j % 16] = 64      # 1 = 64 * 2^-6
        assert torch.equal(k.cpu()[:, 0, :, 0].long(), want) and torch.equal(k, v)
        touched = (want == 64).any(1)
        assert torch.equal(ke.cpu()[:, 0, 0] == 121, touched)


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'int8'])
@pytest.mark.parametrize('D, H, page', [(64, 4, 64), (48, 3, 16), (128, 1, 256), (8, 2, 32), (104, 5, 64)])
def test_read_against_the_pool(D, H, page, kind):
    from streamvoxel_amd.stream.paged import paged_read
    lengths = [0, 1, 15, 64, 65, 700, 33]
    pool = pool_of(kind, lengths, H, D, page, D, token_major=page == 64)
    rows = [pool.rows(b) for b in range(len(lengths))]
    for n, before in ((1, 0), (40, 0), (40, 7), (800, 0), (0, 0)):
        got = paged_read(*pool.args(), n, before=before, **pool.exponents())
        for b, L in enumerate(lengths):
            for t, x in zip(got, rows[b]):
                want = torch.zeros(H, n, D, dtype=torch.float64)
                end = max(0, L - before)
                m = min(n, end)
                want[:, n - m:] = x[:, end - m:end]
                assert torch.equal(t[b].cpu().double(), want), (b, n, before)
    cu = [2]
    for L in lengths:
        cu.append(cu[-1] + min(L, 200))
    T = cu[-1] + 3
    out = [torch.full((T, 2, H, D), 5.0, dtype=torch.bfloat16, device=DEV)[:, i].transpose(0, 1) for i in (0, 1)]
    both = torch.full((T, 2, H, D), 5.0, dtype=torch.bfloat16, device=DEV)
    out = both[:, 0].transpose(0, 1), both[:, 1].transpose(0, 1)       # a token's keys beside its values
    got = paged_read(*pool.args(), T, cu_keys=torch.tensor(cu, dtype=torch.int32, device=DEV), out=out, **pool.exponents())
    for b, L in enumerate(lengths):
        for t, x in zip(got, rows[b]):
            assert torch.equal(t[:, cu[b]:cu[b + 1]].cpu().double(), x[:, L - min(L, 200):])
    assert (both[:2] == 5).all() and (both[cu[-1]:] == 5).all() and got[0] is out[0]


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'int8'])
def test_read_of_bad_pages_is_zeros(kind):
    from streamvoxel_amd.stream.paged import paged_read
    pool = pool_of(kind, [100], 2, 64, 16, 1, clean=True)
    k, v, table, L = pool.args()
    table[0, 3] = pool.pages
    table[0, 5] = -7
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = paged_read(k, v, table, L, 100, bad=bad, **pool.exponents())
    assert int(bad) == 1
    for t, x in zip(got, pool.rows(0)):
        x = x.clone()
        x[:, 48:64] = x[:, 80:96] = 0
        assert torch.equal(t[0].cpu().double(), x)
    bad.zero_()
    got = paged_read(k, v, table[:, :3].contiguous(), L, 100, bad=bad, **pool.exponents())
    assert int(bad) == 1 and not got[0][0, :, 48:].any()
    assert torch.equal(got[0][0, :, :48].cpu().double(), pool.rows(0)[0][:, :48])


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'int8'])
def test_a_sequence_in_chunks_and_tokens(kind):
    """The run that a program makes: queries and keys normed and turned, keys and values held, attention through a window;
    a prompt in two chunks and tokens behind it, against float64 over what the cache then holds, which is read back."""
    from streamvoxel_amd.stream.paged import PagedContext
    from streamvoxel_amd.stream.rotary import norm_rotary, rotary_frequencies
    B, H, Hk, D, W, S = 3, 8, 2, 64, 100, 4
    g = torch.Generator().manual_seed(5)
    freq, amplitude = rotary_frequencies(D, device=DEV)
    wq, wk = [(1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).to(DEV) for _ in 'qk']
    ctx = PagedContext(1, B, Hk, D, 40, DEV, page_size=32, kv_dtype=kind, **(dict(block=16) if kind == 'int8' else {}))
    for n in (130, 61, 1, 1, 1, 7, 1):
        rows = torch.randn(B, n, H + 2 * Hk, D, generator=g).to(torch.bfloat16).to(DEV)
        q, k, v = [t.transpose(1, 2) for t in rows.split((H, Hk, Hk), 2)]
        positions = torch.arange(n, device=DEV) + ctx.host_lengths[0]
        q, k = norm_rotary(q, k, wq, wk, positions, freq, amplitude=amplitude)
        ctx.grow(n)
        ctx.append(0, k, v)
        out = ctx.attend(0, q, causal=True, window=W, sinks=S)
        for b in range(B):
            keys, values = ctx.read(0, b)
            L = ctx.host_lengths[b]
            assert keys.shape == (Hk, L, D)
            want, err = attend64(q[b].cpu().double(), keys.cpu().double(), values.cpu().double(), visible(L, n, True, W, S), D ** -0.5)
            assert ((out[b].cpu().double() - want).abs() <= err).all()
            last = ctx.read(0, b, n=n)
            new = [t[b].cpu().double() for t in (k, v)]
            for mine, t in zip(last, new):
                # Half a step: of e4m3, 2^-4 of the row's largest; of int8, half of 2 / 127 of the largest that the window has.
                step = dict(bf16=0.0, fp8=2.0 ** -4, int8=1 / 127)[kind]
                held = (keys if t is new[0] else values).cpu().double()
                scale = held.abs().amax() if kind == 'int8' else t.abs().amax(-1, keepdim=True)
                assert ((mine.cpu().double() - t).abs() <= step * scale).all()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='capture'), torch.cuda.graph(graph):
        ctx.read(0)
    every = ctx.read(0)
    assert every[0].shape == (Hk, sum(ctx.host_lengths), D) and int(ctx.bad) == 0
    L = ctx.host_lengths[0]
    assert torch.equal(every[0][:, L:2 * L], ctx.read(0, 1)[0])


def test_pools_past_32_bit_offsets():
    """Pages more than 2^32 bytes into the pool, written by the append, read by the attention, with a window and without, and
    read back."""
    from streamvoxel_amd.stream.paged import paged_append, paged_attention, paged_read
    heads, D, page, block = 8, 128, 64, 32
    pages = (1 << 32) // (heads * D * page) + 40
    k, v = [torch.empty(pages, heads, page, D, dtype=torch.int8, device=DEV) for _ in 'kv']
    e = {n: torch.empty(pages, heads, page // block, dtype=torch.uint8, device=DEV) for n in ('k_exponents', 'v_exponents')}
    table = torch.tensor([[pages - 1, 0, pages - 20], [pages - 2, pages - 3, 1]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([180, 129], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(0)
    key, value = [torch.randn(2, heads, 180, D, generator=g).to(torch.bfloat16).to(DEV) for _ in 'kv']
    for b, n in ((0, 180), (1, 129)):
        paged_append(key[b:b + 1, :, :n], value[b:b + 1, :, :n], k, v, table[b:b + 1], lengths[b:b + 1], **e)
    small = Int8Pool([180, 129], heads, D, page, 0, block)
    used = table.flatten().long()
    small.table = torch.arange(6, dtype=torch.int32).view(2, 3)
    small.k, small.v = k[used].cpu(), v[used].cpu()
    small.ke, small.ve = e['k_exponents'][used].cpu(), e['v_exponents'][used].cpu()
    for n in (1, 90):
        q = queries(2, heads, n, D, n)
        for how in (dict(window=None), dict(window=70, sinks=3)):
            check(paged_attention(q, k, v, table, lengths, causal=True, **how, **e), q, small, **how)
    got = paged_read(k, v, table, lengths, 129, **e)
    for b in (0, 1):
        for t, x in zip(got, small.rows(b)):
            assert torch.equal(t[b].cpu().double(), x[:, -129:])
    assert (got[0].float() - torch.stack([key[0, :, 51:], key[1, :, :129]]).float()).abs().max() <= 4 / 127


def test_read_of_more_keys_than_one_launch_holds():
    from streamvoxel_amd.stream.paged import paged_read
    T = (1 << 27) + 9
    pages = -(-T // 1024)
    k, v = [torch.randint(-127, 128, (pages, 1, 1024, 8), device=DEV, dtype=torch.int8) for _ in 'kv']
    e = torch.full((pages, 1, 16), 127, dtype=torch.uint8, device=DEV)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    got = paged_read(k, v, table, torch.tensor([T], dtype=torch.int32, device=DEV), T, k_exponents=e, v_exponents=e)
    for t, pool in zip(got, (k, v)):
        assert torch.equal(t[0, 0].to(torch.int8), pool.view(-1, 8)[:T])


def test_append_of_more_blocks_than_one_launch_holds():
    """More than 2^23 slots of 64 tokens."""
    from streamvoxel_amd.stream.paged import paged_append
    T = (1 << 29) + 70
    pages = -(-T // 1024)
    row = (torch.arange(T, device=DEV) % 127 + 1).to(torch.bfloat16)
    key = row[:, None].expand(T, 8).contiguous()[None, None]
    k, v = [torch.empty(pages, 1, 1024, 8, dtype=torch.int8, device=DEV) for _ in 'kv']
    ke, ve = [torch.zeros(pages, 1, 16, dtype=torch.uint8, device=DEV) for _ in 'kv']
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    paged_append(key, key, k, v, table, torch.tensor([T], dtype=torch.int32, device=DEV), k_exponents=ke, v_exponents=ve)
    assert torch.equal(k.view(-1)[:8 * T].view(torch.int64), v.view(-1)[:8 * T].view(torch.int64)) and torch.equal(ke, ve)
    step = 1 << 26
    for at in list(range(0, T, step)):
        n = min(step, T - at)
        blocks = ke.view(-1)[at // 64:-(-(at + n) // 64)]
        scale = ((blocks.int() << 23).view(torch.float32)).repeat_interleave(64)[:n]
        held = k.view(-1, 8)[at:at + n]
        assert torch.equal(held[:, 0].float() * scale, row[at:at + n].float()), at
        assert (held == held[:, :1]).all(), at


@pytest.mark.parametrize('kind', ['bf16', 'int8'])
def test_captured_calls_follow_lengths_and_contents(kind):
    """Append, reading back and windowed attention in one graph, two graphs with workspaces of their own; several replays
    with the program's eager work between them, each against the eager result."""
    from streamvoxel_amd.stream.paged import paged_append, paged_attention, paged_read
    B, H, Hk, D, page = 5, 8, 2, 64, 64
    g = torch.Generator().manual_seed(3)
    pools = [pool_of(kind, [900, 300, 64, 700, 1], Hk, D, page, 7, clean=True) for _ in 'ab']
    args, es = [list(p.args()) for p in pools], [p.exponents() for p in pools]
    lengths = torch.tensor([800, 200, 60, 600, 1], dtype=torch.int32, device=DEV)
    q, k, v = [torch.zeros(B, n, 1, D, dtype=torch.bfloat16, device=DEV) for n in (H, Hk, Hk)]

    def step(a, e):
        paged_append(k, v, *a[:3], lengths, **e)
        out = paged_attention(q, *a[:3], lengths, causal=True, window=150, sinks=6, **e)
        return out, *paged_read(*a[:3], lengths, 70, **e)

    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(args[0], es[0])
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                static = step(args[0], es[0])
        side.synchronize()
        graphs.append((graph, static))
    fresh = [pool.args() for pool in pools]
    for a, f in zip(args, fresh):
        a[0].copy_(f[0])
        a[1].copy_(f[1])
    for e, pool in zip(es, pools):
        for name, t in pool.exponents().items():
            if t is not None:
                e[name].copy_(t)
    for i in range(6):
        with torch.no_grad():
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g).to(torch.bfloat16) * 2.0 ** (i - 3))
        graph, static = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        want = step(args[1], es[1])
        for a, b in zip(static, want):
            assert torch.equal(a, b), i
        assert torch.equal(args[0][0].view(torch.uint8), args[1][0].view(torch.uint8))
        lengths += 1


def test_engine_over_an_int8_pool():
    """The slot engine's step over int8 pages against the one over bf16 slabs, captured and eager; a slot that is extended; an
    extension that fails leaves the codes as they were.

    A key or value is off by half a step of its block, 2^-8 of the block's largest at most (2^-7 after a growth): the bar is
    that of the e4m3 pool (test_gpu_paged.py), whose values are off by 2^-4 of each."""
    from streamvoxel_amd import synth
    from streamvoxel_amd.stream.engine import Encoded, SlotEngine
    model = synth.StepModel(classes=40, voxel_shape=(64, 16, 16), width=192, depth=4, heads=8, control_width=192,
                            control_depth=2, seed=3)
    for p in model.parameters():
        p.data = p.data.to(torch.bfloat16)
    model = model.to(DEV)
    spec = synth.WindowSpec(height=64, tile=16, num_classes=40)
    make = lambda **kw: SlotEngine(model, spec, DEV, 3, l1_cap=2, l2_cap=8, **kw)
    slab, paged = make(), make(pages=24, page_size=64, kv_dtype='int8')
    assert paged.graph_ok and paged.context.k[0].dtype == torch.int8
    conds = [synth.condition(model, P, L, seed=60 + i, device=DEV) for i, (P, L) in enumerate([(32, 500), (9, 72), (0, 300)])]
    for engine in (slab, paged):
        for i, c in enumerate(conds):
            engine.load_slot(i, c)
        engine.wait_loads()
    with torch.inference_mode():
        want = slab.replay(0.5).patches.float()
        for got in (paged.replay(0.5).patches.float(), paged.eager(0.5).patches.float()):
            assert (got - want).abs().max() <= 2 * 5e-2 * want.abs().max()
            assert (got - want).abs().mean() <= 1e-2 * want.abs().max()
        assert torch.equal(paged.replay(0.5).patches, paged.eager(0.5).patches)
    local, positions = conds[2].local, conds[2].positions
    whole = [paged.context.read(layer, 2) for layer in range(2)]
    paged.load_slot(2, Encoded(conds[2].prefix, local[:, :111], positions[:, :111]))
    paged.wait_loads()

    def failing(*args):
        raise RuntimeError('the layer fails')
    before = [t.clone() for pool in (paged.context.k, paged.context.v, paged.context.k_exponents) for t in pool]
    hook = model.cross[-1].key_value.register_forward_pre_hook(failing)
    with pytest.raises(RuntimeError):
        paged.extend_slot(2, local[:, 111:], positions[:, 111:])
    hook.remove()
    paged.wait_loads()
    after = [t for pool in (paged.context.k, paged.context.v, paged.context.k_exponents) for t in pool]
    assert all(torch.equal(a, b) for a, b in zip(before, after)) and paged.context.host_lengths == [532, 81, 111]
    paged.extend_slot(2, local[:, 111:], positions[:, 111:])
    paged.wait_loads()
    assert paged.packed.lengths.tolist() == [532, 81, 300] and int(paged.context.bad) == 0
    for layer in range(2):
        for a, b in zip(whole[layer], paged.context.read(layer, 2)):
            # (A projection of fewer rows may round differently, by half a step of bf16 each; two roundings of a step at most.)
            scale = a.float().abs().amax((1, 2), keepdim=True)
            assert ((a.float() - b.float()).abs() <= (2 * 2.0 ** -6 + 2 * 2.0 ** -8) * scale).all()


def test_refusals():
    from streamvoxel_amd.stream.paged import PagedContext, paged_append, paged_attention, paged_read
    pool = Int8Pool([100], 2, 64, 64, 1, 32)
    k, v, table, L = pool.args()
    e = pool.exponents()
    q, x = queries(1, 4, 1, 64, 1), queries(1, 2, 1, 64, 1)
    for call in (lambda **how: paged_attention(q, k, v, table, L, **how), lambda **how: paged_read(k, v, table, L, 3, **how),
                 lambda **how: paged_append(x, x, k, v, table, L, **how)):
        with pytest.raises(ValueError, match='exponents'):
            call()
        with pytest.raises(ValueError, match='exponents'):
            call(k_exponents=e['k_exponents'], v_exponents=e['v_exponents'].int())
        with pytest.raises(ValueError, match='alike'):
            call(k_exponents=e['k_exponents'], v_exponents=e['v_exponents'][:, :, :1])
        for blocks in (8, 3):
            wrong = torch.zeros(pool.pages, 2, blocks, dtype=torch.uint8, device=DEV)
            with pytest.raises(ValueError, match='16, 32 or 64'):
                call(k_exponents=wrong, v_exponents=wrong.clone())
    with pytest.raises(ValueError, match='share'):
        paged_append(x, x, k, v, table, L, k_exponents=e['k_exponents'], v_exponents=e['k_exponents'])
    for how in (dict(window=10), dict(window=0, causal=True), dict(window=5, sinks=-1, causal=True), dict(sinks=3, causal=True)):
        with pytest.raises(ValueError, match='window'):
            paged_attention(q, k, v, table, L, **how, **e)
    out = torch.empty(1, 2, 3, 64, dtype=torch.bfloat16, device=DEV)
    for bad in ((out, out), (out, out.float()), (out, out[:, :, :2]), (out, out[:, :1].expand(1, 2, 3, 64))):
        with pytest.raises(ValueError, match='out'):
            paged_read(k, v, table, L, 3, out=bad, **e)
    with pytest.raises(ValueError, match='count'):
        paged_read(k, v, table, L, -1, **e)
    odd = torch.empty(1, 2, 3, 68, dtype=torch.bfloat16, device=DEV)[..., 2:66]
    with pytest.raises(RuntimeError, match='16-byte'):
        paged_read(k, v, table, L, 3, out=(odd, out), **e)
    for how in (dict(kv_dtype='int4'), dict(kv_dtype='int8', block=8), dict(kv_dtype='int8', block=64, page_size=32),
                dict(kv_dtype='fp8', block=16)):
        with pytest.raises(ValueError):
            PagedContext(1, 1, 2, 64, 4, DEV, **how)
