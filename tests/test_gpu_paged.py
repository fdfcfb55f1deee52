"""The append to a paged cache and the attention over it on the GPU, against plain float64 on the host.

Tolerances. Append, bf16: exact for values and unrotated keys; a rotated key is off by the fp32 rotation's 8 * 2^-24 of
|x_a| + |x_b| (test_gpu_rotary.py) and half a step of bf16. e4m3: exponents exact, codes off by half a step, 2^-4 of the
value or 2^-10 of the row's power of two below its normal range.
Attention: the weights are rounded to bf16 (half a step, 2^-8, of each) for the second product, and the sum of them may or
may not be: with A = softmax |v| both together are off by at most 2 * 2^-8 A. A score is an fp32 sum of exact products,
off by D 2^-24 of scale sum |q k|, and the exponent's argument and the exponential by 4 * 2^-24 (1 + |score|) more, which
moves the weights of a row by at most twice that, relatively. The result is rounded to bf16, 2^-8 of it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def _case(msg):
    print(f'[gpu-case] {msg}', flush=True)


class Pool:
    """Pages in a scattered order, filled with values (NaN where no window's keys lie, unless `clean`)."""

    def __init__(self, lengths, heads, D, page, seed, kv_dtype='bf16', spare=3, token_major=False, clean=False, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.heads, self.D, self.page, self.fp8 = lengths, heads, D, page, kv_dtype == 'fp8'
        need = [-(-max(L, 0) // page) for L in lengths]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lengths), max(max(need, default=0), 1)), 0, dtype=torch.int32)
        used = torch.zeros(self.pages, page, dtype=torch.bool)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            for j in range(n):
                used[self.table[b, j], :min(page, lengths[b] - j * page)] = True
            at += n
        shape = (self.pages, heads, page, D)
        k, v = torch.randn(shape, generator=g) * spread, torch.randn(shape, generator=g)
        if not clean:
            k[~used[:, None].expand(-1, heads, -1)] = math.nan
            v[~used[:, None].expand(-1, heads, -1)] = math.nan
        self.ke = self.ve = None
        if self.fp8:
            self.k, self.v = [(t * 64).clamp(-448, 448).to(torch.float8_e4m3fn) for t in (k, v)]
            self.ke, self.ve = [torch.randint(119, 123, shape[:3], generator=g).to(torch.uint8) for _ in 'kv']
        else:
            self.k, self.v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        self.token_major = token_major

    def device(self, t):
        """On the GPU, as [pages, heads, page, D] of dense pages or of pages with a token's heads together."""
        if t is None:
            return None
        if not self.token_major or t.dim() != 4:
            return t.to(DEV)
        return t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)

    def args(self):
        return (self.device(self.k), self.device(self.v), self.table.to(DEV),
                torch.tensor(self.lengths, dtype=torch.int32, device=DEV))

    def exponents(self):
        return dict(k_exponents=self.device(self.ke), v_exponents=self.device(self.ve)) if self.fp8 else {}

    def rows(self, b):
        """Keys and values of window b in float64 [heads, L, D]."""
        L = max(self.lengths[b], 0)
        page = self.table[b, :-(-L // self.page)].long()
        out = []
        for t, e in ((self.k, self.ke), (self.v, self.ve)):
            x = t.view(torch.uint8)[page].view(t.dtype).float().double() if self.fp8 else t[page].double()
            if e is not None:
                x = x * 2.0 ** (e[page].double() - 127)[..., None]
            out.append(x.transpose(0, 1).reshape(self.heads, -1, self.D)[:, :L])
        return out


def attend64(q, k, v, causal, scale):
    """(out, allowed error) of one window: q [H, n, D], k, v [heads, L, D] float64."""
    H, n, D = q.shape
    L, G = k.shape[1], H // k.shape[0]
    if L == 0 or n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    s = scale * q @ k.transpose(1, 2)
    off = 2.0 ** -24 * (D * scale * (q.abs() @ k.abs().transpose(1, 2)) + 4 * (1 + s.abs()))
    if causal:
        seen = torch.arange(L) <= (L - n + torch.arange(n))[:, None]
        s = s.masked_fill(~seen, -math.inf)
        off = off.masked_fill(~seen, 0.0)
    w = (s - s.amax(-1, keepdim=True).clamp(min=-1e300)).exp()
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total.clamp(min=1e-300), torch.zeros_like(w))
    out, A = w @ v, w @ v.abs()
    err = (2 * 2.0 ** -8 + 2 * off.amax(-1, keepdim=True)) * A
    return out, err + 2.0 ** -8 * (out.abs() + err)


def check(got, q, pool, causal, cu=None, scale=None):
    """got, q [B, H, n, D] or packed [H, T, D]."""
    scale = 1 / math.sqrt(pool.D) if scale is None else scale
    got, q = got.cpu().double(), q.cpu().double()
    for b in range(len(pool.lengths)):
        cut = (lambda t: t[b]) if cu is None else (lambda t: t[:, cu[b]:cu[b + 1]])
        out, err = attend64(cut(q), *pool.rows(b), causal, scale)
        off = (cut(got) - out).abs()
        assert not torch.isnan(off).any(), b
        assert (off <= err).all(), (b, (off - err).max().item(), off.max().item())


def queries(B, H, n, D, seed, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, n, H, D, generator=g) * spread).to(torch.bfloat16).to(DEV).transpose(1, 2)


LENGTHS = [[0, 1, 15, 16, 17], [63, 64, 65, 31, 33], [500, 129, 0, 700, 128], [3000], [1537, 40, 9000]]


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
@pytest.mark.parametrize('lengths', LENGTHS, ids=lambda x: '-'.join(map(str, x)))
@pytest.mark.parametrize('n, causal', [(1, False), (1, True), (2, True), (7, False), (40, True), (130, True), (130, False)])
@pytest.mark.parametrize('D, H, heads, page', [(64, 4, 4, 64), (48, 6, 2, 16), (128, 8, 1, 32), (96, 3, 3, 128),
                                               (8, 2, 1, 1024), (72, 4, 2, 16)])
def test_attention_against_float64(lengths, n, causal, D, H, heads, page, kv_dtype):
    """Lengths around the tiles' and the pages' ends, empty windows, windows shorter than their tokens (rows that see
    nothing), NaN in every row that holds no key."""
    from streamvoxel_amd.stream.paged import paged_attention
    _case(f'paged attention {lengths} n={n} causal={causal} D={D} H={H}/{heads} page={page} {kv_dtype}')
    pool = Pool(lengths, heads, D, page, sum(lengths) + n, kv_dtype)
    q = queries(len(lengths), H, n, D, n + D)
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = paged_attention(q, *pool.args(), causal=causal, bad=bad, **pool.exponents())
    assert int(bad) == 0
    check(got, q, pool, causal)


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
@pytest.mark.parametrize('counts', [[1, 0, 5, 1, 1, 200, 33], [0, 0, 3], [1, 1, 1, 1], [129, 1]], ids=str)
@pytest.mark.parametrize('D, H, heads, page', [(64, 4, 1, 16), (128, 4, 4, 64), (96, 8, 2, 32)])
def test_packed_queries(counts, D, H, heads, page, kv_dtype):
    """Windows of different token counts, none among them; rows in front of the first border and behind the last stay."""
    from streamvoxel_amd.stream.paged import paged_attention
    _case(f'packed {counts} D={D} H={H}/{heads} page={page} {kv_dtype}')
    lengths = [n + 37 * i for i, n in enumerate(counts)]
    pool = Pool(lengths, heads, D, page, 3, kv_dtype)
    front, behind = 2, 5
    cu = torch.tensor([0] + counts).cumsum(0) + front
    T = int(cu[-1]) + behind
    q = queries(1, H, T, D, 11)[0]
    for causal in (True, False):
        out = torch.full((T, H, D), 3.0, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
        got = paged_attention(q, *pool.args(), cu_queries=cu.to(torch.int32).to(DEV), causal=causal, out=out,
                              **pool.exponents())
        assert got is out
        check(got, q, pool, causal, cu=cu.tolist())
        assert (out[:, :front] == 3).all() and (out[:, T - behind:] == 3).all()


@pytest.mark.parametrize('n', [1, 100])
def test_attention_of_views(n):
    """Pages with a token's heads together, queries and out in wider buffers, a table row wider than the windows need."""
    from streamvoxel_amd.stream.paged import paged_attention
    pool = Pool([300, 77, 1000], 2, 64, 32, 8, token_major=True)
    k, v, table, lengths = pool.args()
    wide = torch.full((3, 99), -7, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    q = torch.randn(3, n, 3, 6, 72, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)[:, :, 1, :, 8:]
    q = q.transpose(1, 2)
    out = torch.zeros(3, n, 6, 68, dtype=torch.bfloat16, device=DEV)
    paged_attention(q, k, v, wide, lengths, out=out[..., 4:].transpose(1, 2), causal=True)
    check(out[..., 4:].transpose(1, 2), q, pool, True)
    assert (out[..., :4] == 0).all()
    odd = torch.randn(3, n, 6, 65, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)[..., 1:]
    odd = odd.transpose(1, 2)                                       # rows off the 16-byte boundaries: copied
    check(paged_attention(odd, k, v, wide, lengths), odd, pool, False)


@pytest.mark.parametrize('n', [1, 3, 64])
def test_sharp_rows_and_score_jumps(n):
    """Scores of standard deviation 30 and 10, one hot key in any place, scale given."""
    from streamvoxel_amd.stream.paged import paged_attention
    pool = Pool([2000, 65, 700], 2, 64, 16, 4, clean=True)
    for hot in (0, 31, 32, 63, 64, 699):
        pool.k[pool.table[2, hot // 16].long(), :, hot % 16] *= 8
    q = queries(3, 4, n, 64, 6, spread=4.0)
    check(paged_attention(q, *pool.args(), scale=0.9), q, pool, False, scale=0.9)
    check(paged_attention(q, *pool.args(), scale=0.3, causal=True), q, pool, True, scale=0.3)


@pytest.mark.parametrize('n', [1, 50])
def test_infinite_and_nan_keys_touch_their_window_alone(n):
    from streamvoxel_amd.stream.paged import paged_attention
    pool = Pool([400, 400, 400], 1, 64, 64, 4, clean=True)
    pool.k[pool.table[1, 3].long(), :, 7] = math.nan
    q = queries(3, 2, n, 64, 6)
    got = paged_attention(q, *pool.args())
    assert torch.isnan(got[1]).all()
    keep = Pool([400, 400, 400], 1, 64, 64, 4, clean=True)
    same = paged_attention(q, *keep.args())
    assert torch.equal(got[0], same[0]) and torch.equal(got[2], same[2])
    check(same, q, keep, False)


def test_windows_share_pages():
    from streamvoxel_amd.stream.paged import paged_attention
    pool = Pool([200, 260], 2, 64, 64, 4)
    pool.table[0, :3] = pool.table[1, :3]
    pool.lengths = [192, 260]
    q = queries(2, 4, 5, 64, 1)
    check(paged_attention(q, *pool.args(), causal=True), q, pool, True)


@pytest.mark.parametrize('n', [1, 70])
@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
def test_bad_pages_read_as_zeros_and_set_the_flag(n, kv_dtype):
    from streamvoxel_amd.stream.paged import paged_attention
    pool = Pool([300, 128, 64], 2, 64, 32, 4, kv_dtype, clean=True)
    q = queries(3, 2, n, 64, 1)
    k, v, table, lengths = pool.args()
    for number in (-1, pool.pages, 2 ** 31 - 1, -2 ** 31):
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        broken = table.clone()
        broken[0, 2] = number
        got = paged_attention(q, k, v, broken, lengths, bad=bad, **pool.exponents())
        assert int(bad) == 1
        zeroed = Pool([300, 128, 64], 2, 64, 32, 4, kv_dtype, clean=True)
        zeroed.k.view(torch.uint8)[zeroed.table[0, 2].long()] = 0
        zeroed.v.view(torch.uint8)[zeroed.table[0, 2].long()] = 0
        check(got, q, zeroed, False)
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = paged_attention(q, k, v, table, lengths + torch.tensor([1000, 0, 0], device=DEV, dtype=torch.int32), bad=bad,
                          **pool.exponents())
    assert int(bad) == 1
    check(got[1:], q[1:], _tail(pool), False)


def _tail(pool):
    rest = Pool.__new__(Pool)
    rest.__dict__.update(pool.__dict__, lengths=pool.lengths[1:], table=pool.table[1:])
    return rest


def test_negative_lengths_count_as_empty():
    from streamvoxel_amd.stream.paged import paged_attention
    pool = Pool([-5, 40], 1, 64, 16, 4)
    for n in (1, 40):
        q = queries(2, 1, n, 64, 1)
        got = paged_attention(q, *pool.args(), causal=True)
        assert (got[0] == 0).all()
        check(got, q, pool, True)


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
def test_pools_past_32_bit_offsets(kv_dtype):
    """Pages more than 2^32 bytes into the pool, written by the append and read by the attention."""
    from streamvoxel_amd.stream.paged import paged_append, paged_attention
    heads, D, page = 8, 128, 64
    pages = (1 << 32) // (heads * D * page * (1 if kv_dtype == 'fp8' else 2)) + 40
    dtype = torch.float8_e4m3fn if kv_dtype == 'fp8' else torch.bfloat16
    k, v = [torch.empty(pages, heads, page, D, dtype=dtype, device=DEV) for _ in 'kv']
    e = {}
    if kv_dtype == 'fp8':
        e = {n: torch.empty(pages, heads, page, dtype=torch.uint8, device=DEV) for n in ('k_exponents', 'v_exponents')}
    table = torch.tensor([[pages - 1, 0, pages - 20], [pages - 2, pages - 3, 1]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([180, 129], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(0)
    key, value = [torch.randn(2, heads, 180, D, generator=g).to(torch.bfloat16).to(DEV) for _ in 'kv']
    for b, n in ((0, 180), (1, 129)):
        paged_append(key[b:b + 1, :, :n], value[b:b + 1, :, :n], k, v, table[b:b + 1], lengths[b:b + 1], **e)
    small = Pool([180, 129], heads, D, page, 0, kv_dtype)
    used = table.cpu().long()
    small.table = torch.arange(6, dtype=torch.int32).view(2, 3)
    take = lambda t: t.view(torch.uint8)[used.flatten().to(DEV)].cpu().view(t.dtype)
    small.k, small.v = take(k), take(v)
    if e:
        small.ke, small.ve = take(e['k_exponents']), take(e['v_exponents'])
    for n in (1, 90):
        q = queries(2, heads, n, D, n)
        check(paged_attention(q, k, v, table, lengths, causal=True, **e), q, small, True)


# -------------------------------------------------------------------------------------------------------- append

def turned64(x, positions, freq, layout, amplitude):
    """(y, fp32 error) of keys [T, H, D] in float64."""
    angle = positions.double()[:, None] * freq
    c, s = (amplitude * angle.cos())[:, None], (amplitude * angle.sin())[:, None]
    half = freq.numel()
    i = torch.arange(half)
    a, b = (i, i + half) if layout == 'half' else (2 * i, 2 * i + 1)
    y, err = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    err[..., a] = err[..., b] = 8 * 2.0 ** -24 * amplitude * (x[..., a].abs() + x[..., b].abs())
    return y, err


def exponent64(bound):
    e = torch.ceil(torch.log2(bound.double() / 448)) + 127
    return e.clamp(1, 254)


def check_rows(got, code, want, err, bound):
    """Rows [T, H, D] of the cache against want (float64) within err before rounding."""
    if code is None:
        assert ((got.double() - want).abs() <= err + 2.0 ** -8 * (want.abs() + err)).all()
        return
    assert torch.equal(code.double(), exponent64(bound))
    scale = 2.0 ** (code.double() - 127)[..., None]
    off = (got.float().double() * scale - want).abs()
    assert (off <= err + torch.maximum(2.0 ** -4 * (want.abs() + err), 2.0 ** -10 * scale)).all()


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
@pytest.mark.parametrize('layout, part', [(None, 0), ('half', 1.0), ('half', 0.6), ('interleaved', 1.0), ('interleaved', 0.3)])
@pytest.mark.parametrize('D, H, page', [(64, 4, 64), (48, 3, 16), (128, 1, 256), (8, 2, 32), (104, 5, 16)])
@pytest.mark.parametrize('counts, packed, before', [([1, 1, 1], False, 0), ([40, 40, 40], False, 7), ([3, 0, 70, 1], True, 0)])
def test_append_against_float64(counts, packed, before, D, H, page, layout, part, kv_dtype):
    from streamvoxel_amd.stream.paged import paged_append
    _case(f'append {counts} packed={packed} before={before} D={D} H={H} page={page} {layout} {part} {kv_dtype}')
    held = [5, 100, 0, 64][:len(counts)]
    lengths = [h + n + before for h, n in zip(held, counts)]
    pool = Pool(lengths, H, D, page, 5, kv_dtype, clean=True)
    k, v, table, dev_lengths = pool.args()
    k0, v0 = k.clone(), v.clone()
    g = torch.Generator().manual_seed(1)
    T = sum(counts)
    extra = 3 if packed else 0                                      # tokens behind the last window
    key, value = [torch.randn(T + extra, H, D, generator=g).to(torch.bfloat16) for _ in 'kv']
    if kv_dtype == 'fp8':
        key[0], value[T // 2] = 0, 0
        key[T - 1] *= 2.0 ** 100
        value[T - 1] *= 2.0 ** -90
    kw, amplitude = dict(pool.exponents()), 1.0
    explicit = page == 16
    where = torch.cat([torch.arange(L - before - n, L - before) for L, n in zip(lengths, counts)])
    b = torch.cat([torch.full((n,), i) for i, n in enumerate(counts)])
    positions = where
    if layout:
        pairs = max(1, int(D * part) // 2)
        freq = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
        amplitude = 1.2
        kw.update(frequencies=freq.to(DEV), layout=layout, amplitude=amplitude)
        if explicit:
            positions = torch.randint(0, 5000, (T + extra,), generator=g)
            kw['positions'] = positions.to(DEV) if packed else positions.view(len(counts), -1).to(torch.int32).to(DEV)
            positions = positions[:T]
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    dev = lambda t: t.to(DEV).transpose(0, 1) if packed else t.view(len(counts), -1, H, D).to(DEV).transpose(1, 2)
    if packed:
        kw['cu_tokens'] = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(DEV)
    paged_append(dev(key), dev(value), k, v, table, dev_lengths, before=before, bad=bad, **kw)
    assert int(bad) == 0
    page_no, row = table.cpu().long()[b, where // page], where % page
    x, y = key[:T].double(), value[:T].double()
    err = torch.zeros_like(x)
    reach = 1.0
    if layout:
        x, err = turned64(x, positions, freq, layout, amplitude)
        reach = torch.tensor(1.5 * 1.2, dtype=torch.float32)
    at = lambda t: t.view(torch.uint8).cpu().view(t.dtype)[page_no, :, row] if t.dtype != torch.float8_e4m3fn else (
        t.view(torch.uint8).cpu()[page_no, :, row].view(torch.float8_e4m3fn))
    code = (lambda t: t.cpu()[page_no, :, row]) if kv_dtype == 'fp8' else (lambda t: None)
    check_rows(at(k), code(kw.get('k_exponents')) if kv_dtype == 'fp8' else None, x, err,
               key[:T].float().abs().amax(-1) * reach)
    check_rows(at(v), code(kw.get('v_exponents')) if kv_dtype == 'fp8' else None, y, torch.zeros_like(y),
               value[:T].float().abs().amax(-1))
    # Every other row stays.
    mine = torch.zeros(pool.pages, page, dtype=torch.bool)
    mine[page_no, row] = True
    for now, then in ((k, k0), (v, v0)):
        same = (now.view(torch.uint8) == then.view(torch.uint8)).view(pool.pages, H, page, -1).all(-1).cpu()
        assert same[~mine[:, None].expand(-1, H, -1)].all()


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
@pytest.mark.parametrize('D', [48, 96])
def test_axial_append_has_the_bits_of_the_axial_rotation(D, kv_dtype):
    from streamvoxel_amd.stream.paged import paged_append
    from streamvoxel_amd.stream.producer import axial_rope, rope_frequencies
    H, n = 3, 77
    g = torch.Generator().manual_seed(2)
    key, value = [torch.randn(2, n, H, D, generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2) for _ in 'kv']
    positions = (torch.rand(2, n, 3, generator=g) * 64 - 8).to(DEV)
    freq = rope_frequencies(D, device=DEV)
    turned = axial_rope(key, positions, freq)
    results = []
    for how in (dict(positions=positions, frequencies=freq, layout='axial'), {}):
        pool = Pool([n, n + 20], H, D, 32, 1, kv_dtype, clean=True)
        k, v, table, lengths = pool.args()
        e = pool.exponents()
        paged_append(key if how else turned, value, k, v, table, lengths, **how, **e)
        results.append((k, v, e))
    (k, v, e), (k2, v2, e2) = results
    if kv_dtype == 'bf16':
        assert torch.equal(k, k2) and torch.equal(v, v2)
    else:                                # the exponents of rotated keys are chosen before the rotation, and one larger
        value_of = lambda t, x: t.float() * 2.0 ** (x.float() - 127)[..., None]
        a, c = value_of(k, e['k_exponents']), value_of(k2, e2['k_exponents'])
        step = 2.0 ** (e['k_exponents'].float() - 127)[..., None]
        assert ((a - c).abs() <= torch.maximum(2 * 2.0 ** -4 * c.abs(), 2 * 2.0 ** -10 * step)).all()
        assert torch.equal(v.view(torch.uint8), v2.view(torch.uint8))


def test_append_outside_the_table_or_the_pool_writes_nothing():
    from streamvoxel_amd.stream.paged import paged_append
    pool = Pool([64, 64], 2, 64, 32, 1, clean=True)
    k, v, table, lengths = pool.args()
    key = torch.randn(2, 2, 4, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)
    for b, number in ((0, -1), (1, pool.pages), (0, 2 ** 31 - 1), (1, -2 ** 31)):
        k1, v1, broken, bad = k.clone(), v.clone(), table.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
        broken[b, 1] = number
        paged_append(key, key, k1, v1, broken, lengths, bad=bad)
        assert int(bad) == 1
        where = table[b, 1].long()
        assert torch.equal(k1[where], k[where]) and torch.equal(v1[where], v[where])
        other = table[1 - b, 1].long()
        assert torch.equal(k1[other][:, 28:], key[1 - b])
    for off in (40, -64, -62):                                      # past the row's end, and in front of its first key
        k1, v1, bad = k.clone(), v.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
        paged_append(key, key, k1, v1, table, lengths + off, bad=bad)
        assert int(bad) == 1
        assert off == -62 or (torch.equal(k1, k) and torch.equal(v1, v))


def test_append_of_views_and_odd_alignments():
    from streamvoxel_amd.stream.paged import paged_append
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(2, 30, 2, 3, 65, generator=g).to(torch.bfloat16).to(DEV)
    for cut in (slice(0, 64), slice(1, 65)):
        key, value = rows[:, :, 0, :, cut].transpose(1, 2), rows[:, :, 1, :, cut].transpose(1, 2)
        pool = Pool([40, 30], 3, 64, 16, 1, token_major=True, clean=True)
        k, v, table, lengths = pool.args()
        paged_append(key, value, k, v, table, lengths)
        for b, L in ((0, 40), (1, 30)):
            at = torch.arange(L - 30, L, device=DEV)
            page = table[b].long()[at // 16]
            assert torch.equal(k[page, :, at % 16], key[b].transpose(0, 1))
            assert torch.equal(v[page, :, at % 16], value[b].transpose(0, 1))


def test_paged_refusals_on_the_gpu():
    from streamvoxel_amd.stream.paged import paged_append, paged_attention
    pool = Pool([40, 30], 2, 64, 16, 1, clean=True)
    k, v, table, lengths = pool.args()
    key, q = queries(2, 2, 3, 64, 0), queries(2, 4, 3, 64, 0)
    f = torch.ones(32, dtype=torch.float64, device=DEV)
    cu = torch.tensor([0, 3, 6], dtype=torch.int32, device=DEV)
    e8 = dict(k_exponents=torch.zeros(k.shape[:3], dtype=torch.uint8, device=DEV),
              v_exponents=torch.zeros(k.shape[:3], dtype=torch.uint8, device=DEV))
    append = lambda **kw: paged_append(**{**dict(key=key, value=key, k_pages=k, v_pages=v, page_table=table,
                                                 lengths=lengths), **kw})
    attend = lambda **kw: paged_attention(**{**dict(query=q, k_pages=k, v_pages=v, page_table=table, lengths=lengths), **kw})
    for kw in (dict(v_pages=v[:1]), dict(k_pages=k[0], v_pages=v[0]), dict(page_table=table.long()),
               dict(page_table=table.t().contiguous().t()), dict(lengths=lengths.long()), dict(lengths=lengths[:1]),
               dict(bad=torch.zeros(2, dtype=torch.int32, device=DEV)),
               dict(k_pages=k.to(torch.float8_e4m3fn), v_pages=v.to(torch.float8_e4m3fn)),
               dict(k_pages=k.transpose(2, 3), v_pages=v.transpose(2, 3))):
        for call in (append, attend):
            with pytest.raises(ValueError):
                call(**kw)
    for kw in (e8, dict(k_pages=k.float(), v_pages=v.float())):
        for call in (append, attend):
            with pytest.raises(TypeError):
                call(**kw)
    for kw in (dict(value=key[:, :, :2]), dict(key=key[:1], value=key[:1]), dict(key=key[0], value=key[0]), dict(before=-1),
               dict(key=key[:, :1], value=key[:, :1]), dict(cu_tokens=cu), dict(key=key[0], value=key[0], cu_tokens=cu[:2]),
               dict(positions=torch.zeros(2, 3, dtype=torch.int32, device=DEV)), dict(frequencies=f.float()),
               dict(frequencies=f, layout='diagonal'), dict(frequencies=torch.cat((f, f))), dict(frequencies=f[:0]),
               dict(frequencies=f, positions=torch.zeros(2, 4, dtype=torch.int32, device=DEV)),
               dict(frequencies=f, positions=torch.zeros(2, 3, device=DEV)),
               dict(frequencies=f[:10].float(), layout='axial')):
        with pytest.raises(ValueError):
            append(**kw)
    for kw in (dict(query=q[:1]), dict(query=q[..., :48]), dict(query=q[:, :3]), dict(query=q[0]), dict(cu_queries=cu),
               dict(query=q[0], cu_queries=cu.long()), dict(out=q[:, :2]), dict(out=q.float())):
        with pytest.raises(ValueError):
            attend(**kw)
    with pytest.raises(TypeError):
        attend(query=q.float())
    with pytest.raises(TypeError):
        append(key=key.float(), value=key.float())
    with pytest.raises(RuntimeError, match='scale'):
        attend(scale=0.0)


@pytest.mark.parametrize('n', [1, 60])
def test_calls_on_two_streams_and_in_a_graph(n):
    """Two streams at once, and a captured append and attention replayed between eager calls of other sizes."""
    from streamvoxel_amd.stream.paged import paged_append, paged_attention
    g = torch.Generator().manual_seed(6)
    pool = Pool([3000, 200, 1500], 2, 64, 64, 4, clean=True)
    k, v, table, lengths = pool.args()
    q, key = queries(3, 4, n, 64, 1), queries(3, 2, n, 64, 2)
    f = torch.ones(32, dtype=torch.float64, device=DEV) / 100

    def step():
        paged_append(key, key, k, v, table, lengths, frequencies=f)
        return paged_attention(q, k, v, table, lengths, causal=True)
    want = step().clone()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                results.append(paged_attention(q, k, v, table, lengths, causal=True))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        key.copy_(queries(3, 2, n, 64, 20 + i))
        lengths.copy_(torch.tensor([3000 - 100 * i, 200 - i, 1500 + i], dtype=torch.int32))
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            paged_attention(queries(2, 2, 9, 64, i), k, v, table[:2], lengths[:2])
            assert torch.equal(got, step())


# ------------------------------------------------------------------------------------------------ together, in use

@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_a_sequence_in_chunks_and_tokens(kv_dtype, layout):
    """Rotated queries over a cache that grows by chunks and single tokens, against float64 attention of the whole sequences.
    On top of the attention's own error: rotated queries and keys are rounded once (bf16 2^-8; an e4m3 key and value 2^-4 of
    itself or 2^-10 of its row's power of two). A score is then off by scale times the queries' and keys' errors against
    each other, which moves the weights of a row by twice the largest of its row, and a value enters with its own."""
    from streamvoxel_amd.stream.paged import PagedContext
    from streamvoxel_amd.stream.rotary import rotary, rotary_frequencies
    H, heads, D, lengths = 4, 2, 64, [90, 33]
    freq, amplitude = rotary_frequencies(48, scaling='wavelength', factor=4.0, original_length=64, device=DEV)
    ctx = PagedContext(1, 2, heads, D, pages=12, device=DEV, page_size=16, kv_dtype=kv_dtype)
    g = torch.Generator().manual_seed(8)
    q, k, v = [torch.randn(2, n, 90, D, generator=g).to(torch.bfloat16) for n in (H, heads, heads)]
    chunks = [(30, 10), (1, 1), (40, 0), (1, 1), (1, 1), (16, 19), (1, 1)]
    done = [0, 0]
    got = [[], []]
    for counts in chunks:
        ctx.grow(counts)
        cut = lambda t, b: t[b, :, done[b]:done[b] + counts[b]]
        pack = lambda t: torch.cat([cut(t, 0), cut(t, 1)], 1).to(DEV)
        cu = torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32, device=DEV)
        where = torch.cat([torch.arange(done[b], done[b] + counts[b]) for b in range(2)]).to(DEV)
        how = dict(frequencies=freq, layout=layout, amplitude=amplitude)
        ctx.append(0, pack(k), pack(v), cu_tokens=cu, **how)
        turned = rotary(pack(q)[None], where, freq, layout, amplitude)[0]
        out = ctx.attend(0, turned, cu_queries=cu, causal=True)
        for b, o in enumerate(out.split(list(counts), 1)):
            got[b].append(o)
        done = [d + c for d, c in zip(done, counts)]
    assert ctx.host_lengths == ctx.lengths.tolist() == done and int(ctx.bad) == 0
    for b, L in enumerate(done):
        out = torch.cat(got[b], 1).cpu().double()
        where = torch.arange(L)
        tq, eq = turned64(q[b, :, :L].transpose(0, 1).double(), where, freq.cpu(), layout, amplitude)
        tk, ek = turned64(k[b, :, :L].transpose(0, 1).double(), where, freq.cpu(), layout, amplitude)
        value = v[b, :, :L].double()
        eq = (eq + 2.0 ** -8 * (tq.abs() + eq)).transpose(0, 1)
        if kv_dtype == 'bf16':
            ek, ev = ek + 2.0 ** -8 * (tk.abs() + ek), torch.zeros_like(value)
        else:
            step = lambda x, reach: 2.0 ** -10 * 2.0 ** (exponent64(reach * x.float().abs().amax(-1)) - 127)[..., None]
            ek = ek + torch.maximum(2.0 ** -4 * (tk.abs() + ek), step(k[b, :, :L].transpose(0, 1), 1.5 * amplitude))
            ev = torch.maximum(2.0 ** -4 * value.abs(), step(v[b, :, :L], 1.0))
        tq, tk, ek = tq.transpose(0, 1), tk.transpose(0, 1), ek.transpose(0, 1)
        ref, err = attend64(tq, tk, value, True, D ** -0.5)
        G = H // heads
        wide = lambda t: t.repeat_interleave(G, 0)
        ds = D ** -0.5 * (eq @ wide(tk).abs().transpose(1, 2) + (tq.abs() + eq) @ wide(ek).transpose(1, 2))
        seen = torch.ones(L, L, dtype=torch.bool).tril()
        s = (D ** -0.5 * tq @ wide(tk).transpose(1, 2)).masked_fill(~seen, -math.inf)
        most = (ds * seen).amax(-1, keepdim=True)
        moved = torch.expm1(2 * most)                                 # e^(2 ds) bounds a weight's change, sum and all
        A = s.softmax(-1) @ wide(value).abs()
        err = err * (1 + moved) + (moved * A + (1 + moved) * (s.softmax(-1) @ wide(ev))) * (1 + 2.0 ** -6)
        assert ((out - ref).abs() <= err).all(), ((out - ref).abs() - err).max().item()


def _contexts(kv_dtype, batch, pages, **kw):
    from streamvoxel_amd.stream.paged import PagedContext
    from streamvoxel_amd.stream.step import CachedContext
    return (CachedContext(2, batch, 4, 48, 700, DEV, kv_dtype),
            PagedContext(2, batch, 4, 48, pages, DEV, kv_dtype=kv_dtype, **kw))


def test_paged_context_holds_what_the_cached_context_holds():
    """Windows written through both hold the same bits (bf16), also in pages that another window gave back; the attention of
    either is within its bar of float64 over them."""
    from streamvoxel_amd.stream.producer import rope_frequencies
    slab, paged = _contexts('bf16', 3, 30, page_size=16)
    freq = rope_frequencies(48, device=DEV)
    g = torch.Generator().manual_seed(3)
    for P, L, index in ((100, 77, 0), (0, 130, 1), (64, 0, 2), (16, 201, 0), (0, 0, 1), (31, 40, 1)):
        for layer in range(2):
            rows = lambda n: torch.randn(n, 4, 48, generator=g).to(torch.bfloat16).to(DEV).transpose(0, 1)
            pk, pv, k, v = rows(P), rows(P), rows(L), rows(L)
            positions = (torch.rand(L, 3, generator=g) * 60 - 8).to(DEV)
            for ctx in (slab, paged):
                ctx.write(layer, index, k, v, prefix=(pk, pv) if P else None, positions=positions, frequencies=freq)
    assert paged.lengths.tolist() == slab.lengths.tolist() == [217, 71, 64] and int(paged.bad) == 0
    assert paged.free_pages == 30 - 14 - 5 - 4
    for layer in range(2):
        pool = Pool.__new__(Pool)
        pool.__dict__.update(lengths=paged.lengths.tolist(), heads=4, D=48, page=16, fp8=False, ke=None, ve=None,
                             k=paged.k[layer].cpu(), v=paged.v[layer].cpu(), table=paged.table.cpu())
        for b, L in enumerate(pool.lengths):
            k, v = pool.rows(b)
            assert torch.equal(k, slab.k[layer][b, :, :L].cpu().double())
            assert torch.equal(v, slab.vt[layer][b, :, :, :L].transpose(1, 2).cpu().double())
        q = queries(3, 4, 70, 48, layer)
        check(paged.attend(layer, q), q, pool, False)
        check(slab.attend(layer, q), q, pool, False)
        assert torch.equal(paged.attend(layer, q[:2], n=2)[0], paged.attend(layer, q[:2], n=2)[0])


def test_paged_context_errors_leave_it_as_it_was():
    _, paged = _contexts('bf16', 3, 10, page_size=16, max_pages=6)
    paged.resize(0, 70)
    paged.resize(1, 33)
    before = (list(paged.host_lengths), [list(o) for o in paged._owned], paged.free_pages)
    for call, error in ((lambda: paged.resize(2, 97), ValueError), (lambda: paged.resize(2, 40), RuntimeError),
                        (lambda: paged.resize(3, 1), IndexError), (lambda: paged.resize(0, -1), ValueError),
                        (lambda: paged.grow((0, 0)), ValueError), (lambda: paged.grow(30), ValueError),
                        (lambda: paged.grow((0, 30, 30)), RuntimeError)):
        with pytest.raises(error):
            call()
        assert before == (list(paged.host_lengths), [list(o) for o in paged._owned], paged.free_pages)
    paged.release(0)
    paged.resize(2, 96)
    assert paged.lengths.tolist() == [0, 33, 96] and paged.free_pages == 1
    used = [p for own in paged._owned for p in own] + paged._free
    assert sorted(used) == list(range(10))


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
def test_engine_over_a_shared_pool(kv_dtype):
    """The slot engine with pages gives the slab engine's step (captured and eager, over slots of different lengths) up to the
    attention's rounding, holds the same keys, and a slot that is extended holds what a slot loaded whole holds."""
    from streamvoxel_amd import synth
    from streamvoxel_amd.stream.engine import Encoded, SlotEngine
    model = synth.StepModel(classes=40, voxel_shape=(64, 16, 16), width=192, depth=4, heads=8, control_width=192,
                            control_depth=2, seed=3)
    for p in model.parameters():
        p.data = p.data.to(torch.bfloat16)
    model = model.to(DEV)
    spec = synth.WindowSpec(height=64, tile=16, num_classes=40)
    make = lambda **kw: SlotEngine(model, spec, DEV, 3, l1_cap=2, l2_cap=8, kv_dtype=kv_dtype, **kw)
    slab, paged = make(), make(pages=24, page_size=64)
    assert paged.graph_ok and paged.context.max_pages == 10
    conds = [synth.condition(model, P, L, seed=60 + i, device=DEV) for i, (P, L) in enumerate([(32, 500), (9, 72), (0, 300)])]
    for engine in (slab, paged):
        for i, c in enumerate(conds):
            engine.load_slot(i, c)
        engine.wait_loads()
    assert paged.packed.lengths.tolist() == slab.packed.lengths.tolist() == [532, 81, 300]
    with torch.inference_mode():
        want = slab.replay(0.5).patches.float()
        for got in (paged.replay(0.5).patches.float(), paged.eager(0.5).patches.float()):
            # The oracle's bar of the step (test_gpu_forward.py), twice: both engines are within it of the same step.
            bar = 2e-2 if kv_dtype == 'bf16' else 5e-2
            assert (got - want).abs().max() <= 2 * bar * want.abs().max()
            assert (got - want).abs().mean() <= 1e-2 * want.abs().max()
        assert torch.equal(paged.replay(0.5).patches, paged.eager(0.5).patches)
    # The third slot again, its local context in two parts.
    local, positions = conds[2].local, conds[2].positions
    rows = lambda: [t[layer].view(torch.uint8)[paged.context.table[2, :5].long()].clone()
                    for layer in range(2) for t in (paged.context.k, paged.context.v)]
    whole = rows()
    paged.load_slot(2, Encoded(conds[2].prefix, local[:, :111], positions[:, :111]))
    paged.extend_slot(2, local[:, 111:], positions[:, 111:])
    paged.wait_loads()
    assert paged.packed.lengths.tolist() == [532, 81, 300] and int(paged.context.bad) == 0
    # (A projection of fewer rows may round differently: one half step of bf16 against another, and of e4m3 on top.)
    held = lambda t: t.view(torch.bfloat16).float() if kv_dtype == 'bf16' else t.view(torch.float8_e4m3fn).float()
    for a, b in zip(whole, rows()):
        a, b = held(a)[:4], held(b)[:4]
        assert (a - b).abs().max() <= (2.0 ** -5 if kv_dtype == 'bf16' else 2.0 ** -2) * a.abs().max()
        assert (a != b).float().mean() < 0.02
    with pytest.raises(ValueError, match='pages'):
        slab.extend_slot(0, local, positions)
    with pytest.raises(ValueError, match='capacity'):
        paged.extend_slot(0, torch.zeros(1, 200, 192, device=DEV), torch.zeros(1, 200, 3, device=DEV))
    with pytest.raises(IndexError):
        paged.extend_slot(3, local, positions)


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
@pytest.mark.parametrize('D, heads, page', [(64, 1, 64), (128, 2, 16)])
@pytest.mark.parametrize('n, at, packed', [(2, 1, False), (3, 1, False), (16, 9, False), (40, 17, False), (200, 70, False), (200, 199, True),
                                           (32, 1, True)])
def test_what_a_token_does_not_see_does_not_reach_it(n, at, packed, D, heads, page, kv_dtype):
    """A key and a value of the chunk's token `at` that are not finite: the tokens in front of it are as if it were not there,
    it and the later ones have the formula's NaN and infinities."""
    from streamvoxel_amd.stream.paged import paged_attention
    _case(f'values that are not finite: n={n} at={at} packed={packed} D={D} page={page} {kv_dtype}')
    L = 700
    j = L - n + at
    for what in ('v', 'k', 'inf'):
        if what == 'inf' and kv_dtype == 'fp8':
            continue   # (no code for it)
        pool = Pool([900, L], heads, D, page, n + D, kv_dtype, clean=True)
        q = queries(2, 2 * heads, n, D, n)
        row = (pool.table[1, j // page].long(), slice(None), j % page)
        if what == 'k':
            pool.k[row] = torch.full((heads, D), math.nan).to(pool.k.dtype)
        else:
            v = torch.where(torch.arange(D) == 5, math.inf if what == 'inf' else math.nan, pool.v[row].float())
            pool.v[row] = v.to(pool.v.dtype)
        cu, qq = None, q
        if packed:
            cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=DEV)
            qq = torch.cat((q[0], q[1]), 1)
        got = paged_attention(qq, *pool.args(), cu_queries=cu, causal=True, **pool.exponents())
        if packed:
            got = torch.stack((got[:, :n], got[:, n:]))
        k, v = pool.rows(1)
        want, err = attend64(q[1, :, :at].cpu().double(), k[:, :j], v[:, :j], True, D ** -0.5)
        assert ((got[1, :, :at].cpu().double() - want).abs() <= err).all()
        check(got[:1], q[:1], _window(pool, 0), True)
        late = got[1, :, at:].cpu()
        if what == 'k':
            assert torch.isnan(late).all()
            continue
        assert (torch.isnan if what == 'v' else torch.isposinf)(late[..., 5]).all()
        k, v = k, v.masked_fill(torch.arange(D) == 5, 0.0)
        want, err = attend64(q[1].cpu().double(), k, v, True, D ** -0.5)
        rest = torch.arange(D) != 5
        assert ((late.double() - want[:, at:]).abs() <= err[:, at:])[..., rest].all()


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
@pytest.mark.parametrize('B', [65, 200, 1100])
@pytest.mark.parametrize('kind', ['tokens', 'chunks', 'packed'])
def test_many_windows(kind, B, kv_dtype):
    """More windows than a workgroup plans by itself: short ones, empty ones, a few long enough for parts."""
    from streamvoxel_amd.stream.paged import paged_attention
    _case(f'many windows: {kind} B={B} {kv_dtype}')
    lengths = [(0, 1, 40, 17, 64, 3, 100)[b % 7] if b % 60 != 31 else 900 + b for b in range(B)]
    pool = Pool(lengths, 1, 16, 16, B, kv_dtype)
    if kind != 'packed':
        n = 1 if kind == 'tokens' else 33
        q = queries(B, 2, n, 16, B)
        check(paged_attention(q, *pool.args(), causal=True, **pool.exponents()), q, pool, True)
        return
    counts = [(1, 0, 5, 1, 40, 1, 17)[b % 7] if b % 60 != 31 else (130 if b % 120 == 31 else 1) for b in range(B)]
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    g = torch.Generator().manual_seed(B)
    q = torch.randn(2, cu[-1], 16, generator=g).to(torch.bfloat16).to(DEV)
    got = paged_attention(q, *pool.args(), cu_queries=torch.tensor(cu, dtype=torch.int32, device=DEV), causal=True,
                          **pool.exponents())
    check(got, q, pool, True, cu)
    one = paged_attention(q[:, cu[31]:cu[32]].contiguous(), *[t[31:32] if i > 1 else t for i, t in enumerate(pool.args())],
                          cu_queries=torch.tensor([0, counts[31]], dtype=torch.int32, device=DEV), causal=True,
                          **pool.exponents())
    check(one, q[:, cu[31]:cu[32]], _window(pool, 31), True, [0, counts[31]])


def _window(pool, b):
    kept = Pool.__new__(Pool)
    kept.__dict__.update(pool.__dict__, lengths=pool.lengths[b:b + 1], table=pool.table[b:b + 1])
    return kept


def test_rows_off_their_alignment_are_copied():
    """Contiguous queries, keys and values that start between 16-byte boundaries."""
    from streamvoxel_amd.stream.paged import paged_append, paged_attention
    pool = Pool([40, 30], 2, 64, 16, 1, clean=True)
    k, v, table, lengths = pool.args()
    g = torch.Generator().manual_seed(2)
    flat = torch.randn(2, 2 * 2 * 3 * 64 + 1, generator=g).to(torch.bfloat16).to(DEV)
    key, value = [t[1:].view(2, 2, 3, 64) for t in flat]
    assert key.is_contiguous() and key.data_ptr() % 16
    check(paged_attention(key, k, v, table, lengths), key, pool, False)
    paged_append(key, value, k, v, table, lengths)
    for b, L in ((0, 40), (1, 30)):
        at = torch.arange(L - 3, L, device=DEV)
        page = table[b].long()[at // 16]
        assert torch.equal(k[page, :, at % 16], key[b].transpose(0, 1))
        assert torch.equal(v[page, :, at % 16], value[b].transpose(0, 1))


@pytest.mark.parametrize('n', [1, 50])
def test_out_over_the_query_and_refused_places(n):
    from streamvoxel_amd.stream.paged import paged_append, paged_attention
    pool = Pool([1500, 30], 2, 64, 16, 1, clean=True)
    args = pool.args()
    q = queries(2, 4, n, 64, 3)
    want = paged_attention(q, *args, causal=True)
    over = q.clone(memory_format=torch.preserve_format)
    assert paged_attention(over, *args, causal=True, out=over) is over
    assert torch.equal(over, want)
    room = torch.zeros(2, 4, n + 1, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match='share'):
        paged_attention(room[:, :, :n], *args, out=room[:, :, 1:])
    with pytest.raises(ValueError, match='place'):
        paged_attention(q, *args, out=room[:, :1, :n].expand(2, 4, n, 64))
    key = queries(2, 2, n, 64, 4)
    with pytest.raises(ValueError, match='place'):
        paged_append(key, key, args[0][:1].expand(args[0].shape), args[1], *args[2:])


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
@pytest.mark.parametrize('page', [16, 64])
@pytest.mark.parametrize('D', range(8, 129, 8))
def test_every_head_width(D, page, kv_dtype):
    """Single tokens, chunks, and both packed, with windows short and long enough for parts."""
    from streamvoxel_amd.stream.paged import paged_append, paged_attention
    _case(f'head width D={D} page={page} {kv_dtype}')
    pool = Pool([700, 90], 2, D, page, D, kv_dtype)
    args, how = pool.args(), dict(causal=True, **pool.exponents())
    for n in (1, 40):
        q = queries(2, 4, n, D, n)
        check(paged_attention(q, *args, **how), q, pool, True)
    cu = [0, 1, 41]
    q = torch.randn(4, 41, D, generator=torch.Generator().manual_seed(D)).to(torch.bfloat16).to(DEV)
    got = paged_attention(q, *args, cu_queries=torch.tensor(cu, dtype=torch.int32, device=DEV), **how)
    check(got, q, pool, True, cu)
    key = queries(2, 2, 3, D, 5)
    paged_append(key, key, *args, **pool.exponents())
    if kv_dtype == 'bf16':
        at = torch.arange(697, 700, device=DEV)
        assert torch.equal(args[0][args[2][0].long()[at // page], :, at % page], key[0].transpose(0, 1))


@pytest.mark.parametrize('B', [20, 90])
def test_a_captured_call_follows_lengths_and_borders(B):
    """A packed call captured once: its plan is made on the device at every replay, whatever the lengths and the borders
    are by then."""
    from streamvoxel_amd.stream.paged import paged_attention
    longest, T = 1200, 400
    pool = Pool([longest] * B, 2, 32, 64, B, clean=True)
    k, v, table, lengths = pool.args()
    q = torch.randn(4, T, 32, generator=torch.Generator().manual_seed(B)).to(torch.bfloat16).to(DEV)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    call = lambda: paged_attention(q, k, v, table, lengths, cu_queries=cu, causal=True)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    g = torch.Generator().manual_seed(1)
    for most in (30, longest, 1, longest):
        pool.lengths = torch.randint(0, most + 1, (B,), generator=g).tolist()
        cut = sorted(torch.randint(0, T + 1, (B - 1,), generator=g).tolist())
        borders = [0, *cut, T] if most > 1 else [0] * B + [T]
        lengths.copy_(torch.tensor(pool.lengths, dtype=torch.int32))
        cu.copy_(torch.tensor(borders, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check(out, q, pool, True, borders)
        assert torch.equal(out, call())


@pytest.mark.parametrize('kv_dtype, n', [('bf16', 5), ('fp8', 17)])
@pytest.mark.parametrize('times', [1, 2])
def test_a_long_window_among_tiles_beside_single_tokens(times, kv_dtype, n):
    """Packed windows of both forms, the tiles as many as half of the chip and one window of them cut (test_paged_plan.py: more
    places than a full share): every row is written, by its window's keys."""
    from streamvoxel_amd.stream.paged import paged_attention
    _case(f'a long window beside single tokens: {times} x 60 windows {kv_dtype}')
    heads = 8 // times
    counts = [n] * 52 * times + [1] * 8 * times
    lengths = [64000] + [384] * (52 * times - 1) + [8192] * 8 * times
    pool = Pool(lengths, heads, 16, 64, times, kv_dtype)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    q = torch.randn(heads, cu[-1], 16, generator=torch.Generator().manual_seed(times)).to(torch.bfloat16).to(DEV)
    out = torch.full_like(q, math.nan)
    for causal in (True, False):
        out.fill_(math.nan)
        paged_attention(q, *pool.args(), cu_queries=torch.tensor(cu, dtype=torch.int32, device=DEV), causal=causal, out=out,
                        **pool.exponents())
        check(out, q, pool, causal, cu)


def test_windows_of_one_context_on_two_streams():
    """A window that is written on a side stream, behind other work there, while the others grow on the current one: every
    length and every key is the last call's for its window."""
    from streamvoxel_amd.stream.paged import PagedContext
    ctx = PagedContext(1, 6, 2, 64, 60, DEV, page_size=16)
    g = torch.Generator().manual_seed(5)
    rows = lambda n: torch.randn(2, n, 64, generator=g).to(torch.bfloat16).to(DEV)
    held = [[torch.empty(2, 0, 64, dtype=torch.bfloat16, device=DEV)] for _ in range(6)]
    side, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device=DEV)
    for step, counts in enumerate([(0, 3, 20, 1, 1, 1), (0, 1, 0, 17, 0, 2), (0, 16, 16, 16, 16, 16)]):
        loaded, new = rows(40 + 30 * step), [rows(n) for n in counts]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                busy @ busy
            ctx.resize(0, loaded.shape[1])
            ctx.append(0, loaded, loaded, index=0)
        ctx.grow(counts)
        for b in range(1, 6):
            ctx.append(0, new[b], new[b], index=b)
            held[b].append(new[b])
        held[0] = [loaded]
        torch.cuda.synchronize()
        assert ctx.lengths.tolist() == ctx.host_lengths == [sum(t.shape[1] for t in h) for h in held]
        for b in range(6):
            at = torch.arange(ctx.host_lengths[b], device=DEV)
            page = ctx.table[b].long()[at // 16]
            assert torch.equal(ctx.k[0][page, :, at % 16].transpose(0, 1), torch.cat(held[b], 1)), (step, b)
    assert int(ctx.bad) == 0


def test_pages_that_change_hands_between_streams():
    """A window written on a busy side stream twice, long and then short, while another takes the pages that it gave back: what
    the first write puts there is overwritten by the other window's keys, not they by it."""
    from streamvoxel_amd.stream.paged import PagedContext
    ctx = PagedContext(1, 2, 2, 64, 8, DEV, page_size=16)
    g = torch.Generator().manual_seed(6)
    long, short, other = [torch.randn(2, n, 64, generator=g).to(torch.bfloat16).to(DEV) for n in (128, 16, 112)]
    side, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ctx.resize(0, 128)
        for _ in range(20):
            busy @ busy
        ctx.append(0, long, long, index=0)
        ctx.resize(0, 16)
        ctx.append(0, short, short, index=0)
    ctx.grow((0, 112))
    ctx.append(0, other, other, index=1)
    torch.cuda.synchronize()
    assert ctx.lengths.tolist() == [16, 112] and int(ctx.bad) == 0
    for b, want in ((0, short), (1, other)):
        at = torch.arange(want.shape[1], device=DEV)
        assert torch.equal(ctx.v[0][ctx.table[b].long()[at // 16], :, at % 16].transpose(0, 1), want)


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
def test_an_extension_that_fails_leaves_the_slot_as_it_was(kv_dtype):
    """A local context of the wrong width, and one that fails in the last layer: lengths, pages and the step stay; a good one
    then grows the slot."""
    from streamvoxel_amd import synth
    from streamvoxel_amd.stream.engine import SlotEngine
    model = synth.StepModel(classes=40, voxel_shape=(64, 16, 16), width=192, depth=4, heads=8, control_width=192,
                            control_depth=2, seed=3)
    for p in model.parameters():
        p.data = p.data.to(torch.bfloat16)
    model = model.to(DEV)
    spec = synth.WindowSpec(height=64, tile=16, num_classes=40)
    engine = SlotEngine(model, spec, DEV, 2, l1_cap=2, l2_cap=8, kv_dtype=kv_dtype, pages=24)
    conds = [synth.condition(model, P, L, seed=70 + i, device=DEV) for i, (P, L) in enumerate([(32, 100), (9, 72)])]
    for i, c in enumerate(conds):
        engine.load_slot(i, c)
    engine.wait_loads()
    want, free = engine.replay(0.5).patches.clone(), engine.context.free_pages
    more = synth.condition(model, 0, 90, seed=80, device=DEV)

    def failing(*args):
        raise RuntimeError('the layer fails')
    for break_it in (False, True):
        hook = model.cross[-1].key_value.register_forward_pre_hook(failing) if break_it else None
        with pytest.raises(RuntimeError):
            engine.extend_slot(1, more.local if break_it else more.local[..., 8:], more.positions)
        if hook is not None:
            hook.remove()
        engine.wait_loads()
        assert engine.packed.lengths.tolist() == engine.context.host_lengths == [132, 81]
        assert engine.context.free_pages == free and int(engine.context.bad) == 0
        assert torch.equal(engine.replay(0.5).patches, want)
    engine.extend_slot(1, more.local, more.positions)
    engine.wait_loads()
    assert engine.packed.lengths.tolist() == engine.context.host_lengths == [132, 171]
    assert not torch.equal(engine.replay(0.5).patches, want)


@pytest.mark.parametrize('kv_dtype', ['bf16', 'fp8'])
@pytest.mark.parametrize('n', [1, 40])
@pytest.mark.parametrize('D', [8, 24, 40, 72, 104, 120, 64])
def test_a_key_whose_score_is_minus_infinity_has_no_weight(D, n, kv_dtype):
    """One element of a key infinite against queries of the other sign there, in both forms and at widths whose last step is
    half empty: the formula's finite result. (e4m3 has no code for an infinity: 448 2^127 there.)"""
    from streamvoxel_amd.stream.paged import paged_attention
    pool = Pool([90, 40], 2, D, 16, D, kv_dtype, clean=True)
    q = queries(2, 4, n, D, n)
    q[..., 3] = -q[..., 3].abs() - 0.125
    j = 37
    row = (pool.table[0, j // 16].long(), slice(None), j % 16)
    key = pool.k[row].float()
    if kv_dtype == 'bf16':
        key[:, 3] = math.inf
        pool.k[row] = key.to(pool.k.dtype)
    else:
        key[:], key[:, 3] = 0, 448
        pool.k[row] = key.to(pool.k.dtype)
        pool.ke[row] = 254
    got = paged_attention(q, *pool.args(), **pool.exponents())
    k, v = pool.rows(0)
    keep = [i for i in range(90) if i != j]
    want, err = attend64(q[0].cpu().double(), k[:, keep], v[:, keep], False, D ** -0.5)
    off = (got[0].cpu().double() - want).abs()
    assert not torch.isnan(off).any() and (off <= err).all()
    check(got[1:], q[1:], _window(pool, 1), False)


@pytest.mark.parametrize('n', [1, 50])
def test_odd_strides_of_dimensions_with_one_element(n):
    """One window or one head whose stride, never used, is no multiple of 8: taken as it is, or copied where the rows lie
    between 16-byte boundaries too."""
    from streamvoxel_amd.stream.paged import paged_append, paged_attention
    from streamvoxel_amd.stream.rotary import rotary
    pool = Pool([400], 1, 64, 16, 1, clean=True)
    k, v, table, lengths = pool.args()
    buffer = torch.randn(70 * 64 + 9, generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).to(DEV)
    f = torch.ones(32, dtype=torch.float64, device=DEV) / 100
    for start, strides in ((0, (n * 64 + 1, 3, 64, 1)), (1, (n * 64 + 1, 5, 64, 1)), (8, (7, n * 64 + 3, 64, 1))):
        x = buffer.as_strided((1, 1, n, 64), strides, start)
        same = x.clone(memory_format=torch.contiguous_format)
        want = paged_attention(same, k, v, table.clone(), lengths, causal=True)
        assert torch.equal(paged_attention(x, k, v, table, lengths, causal=True), want)
        out = torch.zeros(n * 64 + 9, dtype=torch.bfloat16, device=DEV).as_strided((1, 1, n, 64), (n * 64 + 1, 1, 64, 1), 4)
        assert torch.equal(paged_attention(x, k, v, table, lengths, causal=True, out=out), want)
        check(want, same, pool, True)
        pages = [torch.zeros(pool.pages, 16, 64, dtype=torch.bfloat16, device=DEV).as_strided(k.shape, (1024, 3, 64, 1))
                 for _ in 'kv']
        paged_append(x, x, *pages, table, lengths)
        at = torch.arange(400 - n, 400, device=DEV)
        assert torch.equal(pages[0][table[0].long()[at // 16], :, at % 16].transpose(0, 1), same[0])
        turned = rotary(x, torch.arange(n, device=DEV), f)
        assert torch.equal(turned, rotary(same, torch.arange(n, device=DEV), f))


def test_books_do_not_change_in_a_capture():
    """grow, resize and release are refused while their stream is captured; append and attend there are the graph's work."""
    from streamvoxel_amd.stream.paged import PagedContext
    ctx = PagedContext(1, 2, 2, 64, 6, DEV, page_size=16)
    key, q = queries(2, 2, 5, 64, 0), queries(2, 4, 5, 64, 1)
    ctx.grow(5)
    ctx.append(0, key, key)
    want = ctx.attend(0, q, causal=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for change in (lambda: ctx.grow(1), lambda: ctx.release(0), lambda: ctx.resize(1, 40)):
            with pytest.raises(RuntimeError, match='capture'):
                change()
        ctx.append(0, key, key)
        out = ctx.attend(0, q, causal=True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and ctx.lengths.tolist() == ctx.host_lengths == [5, 5] and ctx.free_pages == 4
        ctx.grow(0)


def test_append_of_more_tokens_than_one_launch_holds():
    """More than 2^24 workgroups, which no launch of 256 threads each holds."""
    from streamvoxel_amd.stream.paged import paged_append
    T = (1 << 27) + 9
    pages = -(-T // 1024)
    key = torch.randn(1, 1, T, 8, device=DEV, generator=torch.Generator(DEV).manual_seed(1), dtype=torch.bfloat16)
    k, v = [torch.zeros(pages, 1, 1024, 8, dtype=torch.bfloat16, device=DEV) for _ in 'kv']
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    paged_append(key, key, k, v, table, torch.tensor([T], dtype=torch.int32, device=DEV))
    for t in (k, v):
        assert torch.equal(t.view(-1, 8)[:T], key[0, 0]) and not t.view(-1, 8)[T:].any()


@pytest.mark.parametrize('n', [1, 5])
def test_attention_of_more_windows_than_one_launch_holds(n):
    """More than 2^24 workgroups of either form, all windows over one page."""
    from streamvoxel_amd.stream.paged import paged_attention
    B, D = (1 << 24) + 3, 8
    g = torch.Generator(DEV).manual_seed(n)
    q = torch.randn(B, 1, n, D, device=DEV, generator=g, dtype=torch.bfloat16)
    k, v = [torch.randn(1, 1, 16, D, device=DEV, generator=g, dtype=torch.bfloat16) for _ in 'kv']
    lengths = torch.randint(0, 17, (B,), device=DEV, generator=g, dtype=torch.int32)
    got = paged_attention(q, k, v, torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(B, 1), lengths)
    for L in range(17):
        mine = (lengths == L).nonzero()[:, 0]
        out, err = attend64(q[mine].view(1, -1, D).double(), k[0, :, :L].double(), v[0, :, :L].double(), False, D ** -0.5)
        assert ((got[mine].view(1, -1, D).double() - out).abs() <= err).all(), L


def test_a_join_of_more_rows_than_one_launch_holds():
    """2^27 rows of a window without keys, and behind them a window whose keys are cut: its parts are joined."""
    from streamvoxel_amd.stream.paged import paged_attention
    H, D, first, last, L = 128, 8, 1 << 20, 200, 100000
    g = torch.Generator(DEV).manual_seed(1)
    q = torch.randn(first + last, H, D, device=DEV, generator=g, dtype=torch.bfloat16).transpose(0, 1)
    pages = -(-L // 1024)
    k, v = [torch.randn(pages, 1, 1024, D, device=DEV, generator=g, dtype=torch.bfloat16) for _ in 'kv']
    table = torch.arange(pages, dtype=torch.int32, device=DEV).expand(2, pages)
    out = torch.full_like(q, math.nan)
    paged_attention(q, k, v, table, torch.tensor([0, L], dtype=torch.int32, device=DEV), out=out,
                    cu_queries=torch.tensor([0, first, first + last], dtype=torch.int32, device=DEV))
    assert not out[:, :first].any()
    rows = [t.reshape(1, -1, D)[:, :L].double().cpu() for t in (k, v)]
    for at in (0, 100, last - 2):
        cut = slice(first + at, first + at + 2)
        want, err = attend64(q[:, cut].cpu().double(), *rows, False, D ** -0.5)
        assert ((out[:, cut].cpu().double() - want).abs() <= err).all(), at
