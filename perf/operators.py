"""Rotary positions, the append to a paged cache and the attention over it, in their plain forms and as calls of the
framework.

`listed()` gives the fixed cases and `draw(rng)` further ones of the same ranges; `prepare` makes what a program holds
before the call, `run` makes one pass, `work` counts what the pass cannot do without, `exact` gives the result in 64
bits.
Where `own` is false `run` computes from elementary torch operations, else through streamvoxel_amd.

Layouts: heads before tokens, as the framework's attention takes them ([B, H, n, D], or packed [H, T, D] with the
windows' borders); a pool of pages [pages, heads, page, D] and each window's row of page numbers. An e4m3 pool has one
power of two a row and head, 2^(exponent - 127).
"""
import math
import random

import torch

own = False

DEVICE = 'cuda'
E4M3_MAX = 448.0


def listed():
    return [
        # One new token for each of 64 windows: what latency allows.
        _rotary('rotary_tokens', windows=64, tokens=1, heads=16, head_dim=64, part=64, layout='half', far=131072),
        # The queries of 8 windows as they leave the projection; half of the head turns, positions squeezed by 4.
        _rotary('rotary_chunk', windows=8, tokens=1024, heads=12, head_dim=64, part=32, layout='interleaved', far=9744,
                stretch=4.0),
        # Training on one long sequence in fp32: the rotation and its gradient.
        _rotary('rotary_train', windows=1, tokens=32768, heads=16, head_dim=128, part=128, layout='half', far=32768,
                dtype='fp32', gradient=True, stretch=8.0, amplitude=1.2079441541679836),
        # One new token's keys and values for each of 64 windows.
        _append('append_tokens', windows=64, low=1, high=1, held=512, heads=16, head_dim=64, page=64, turn='half'),
        # A window's local context, three-axis positions, after 4096 keys that are there (the shipped model's heads).
        _append('append_window', windows=1, low=8480, high=8480, held=4096, heads=8, head_dim=48, page=64,
                turn='axial'),
        # A ragged batch of chunks into an e4m3 pool of small pages.
        _append('append_chunks_e4m3', windows=32, low=1, high=1024, held=300, heads=8, head_dim=128, page=16,
                turn='interleaved', cache='fp8', packed=True),
        # One token of one window over all of its context: a lone player's latency.
        _attend('attend_token', windows=1, low=1, high=1, short=9744, long=9744, heads=12, groups=1, head_dim=64,
                page=64),
        # One token of each of 64 windows, four heads to a key head, long contexts.
        _attend('attend_tokens', windows=64, low=1, high=1, short=512, long=16384, heads=16, groups=4, head_dim=128,
                page=64, causal=True),
        # The same over an e4m3 pool, a key head for each head.
        _attend('attend_tokens_e4m3', windows=64, low=1, high=1, short=1552, long=9744, heads=16, groups=1, head_dim=64,
                page=32, causal=True, cache='fp8'),
        # The cross attention of the 8-slot step over a shared pool: 1024 queries a window, every key seen.
        _attend('attend_windows', windows=8, low=1024, high=1024, short=1552, long=9744, heads=12, groups=1,
                head_dim=64, page=64),
        # A chunk of new tokens behind what each of 4 windows holds.
        _attend('attend_chunk', windows=4, low=512, high=512, short=2048, long=16384, heads=16, groups=4, head_dim=128,
                page=128, causal=True),
        # A serving step: a few chunks beside many single tokens, packed, in small pages.
        _attend('attend_mixed', windows=24, low=1, high=512, short=600, long=8192, heads=8, groups=1, head_dim=96,
                page=16, causal=True, packed=True, single=0.75),
    ]


def draw(rng):
    most = {}
    for case in listed():
        w, kind = work(case), case['kind']
        most[kind] = [max(a, w[n]) for a, n in zip(most.get(kind, [0, 0]), ('bytes', 'flops'))]
    while True:
        case = _drawn(rng)
        w = work(case)
        if w['bytes'] <= most[case['kind']][0] and w['flops'] <= most[case['kind']][1] and _padded(case) <= 1 << 31:
            return case


def _padded(case):
    """(query, key) pairs of a batch padded to its longest, which the plain attention holds at once."""
    return case['windows'] * case['heads'] * case['high'] * case['long'] if case['kind'] == 'attend' else 0


def _drawn(rng):
    kind = rng.choice(['rotary', 'append', 'attend', 'attend'])
    head_dim = rng.choice([48, 64, 64, 96, 128])
    if kind == 'rotary':
        head_dim = rng.choice([head_dim, 2 * rng.randint(4, 64)])
        return _rotary(None, windows=_log(rng, 1, 64), tokens=_log(rng, 1, 32768), heads=rng.choice([4, 8, 12, 16, 32]),
                       head_dim=head_dim, part=rng.choice([head_dim, 2 * rng.randint(1, head_dim // 2)]),
                       layout=rng.choice(['half', 'interleaved']), far=_log(rng, 64, 1 << 20),
                       dtype=rng.choice(['bf16', 'bf16', 'fp32']), gradient=rng.random() < 0.3,
                       stretch=rng.choice([1.0, 2.0, 8.0]), amplitude=rng.choice([1.0, 1.0, 1.1]))
    windows, packed, page = _log(rng, 1, 64), rng.random() < 0.4, rng.choice([16, 32, 64, 64, 128, 256])
    cache, pick = rng.choice(['bf16', 'bf16', 'fp8']), rng.randrange(1 << 20)
    if kind == 'append':
        high = rng.choice([1, _log(rng, 2, 8480)])
        turn = rng.choice(['half', 'interleaved', 'none', 'axial' if head_dim % 6 == 0 else 'half'])
        held = rng.choice([0, _log(rng, 1, 4096)])
        return _append(None, windows=windows, low=1 if packed else high, high=high, held=held,
                       heads=rng.choice([1, 2, 4, 8, 12, 16]), head_dim=head_dim, page=page, turn=turn, cache=cache,
                       packed=packed, pick=pick)
    heads = rng.choice([4, 8, 12, 16])
    high = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 2048)])
    long = _log(rng, max(16, high), 16384)
    return _attend(None, windows=windows, low=1 if packed else high, high=high, short=rng.randint(high, long),
                   long=long, heads=heads, groups=rng.choice([1, 1, 2, 4]), head_dim=head_dim, page=page,
                   causal=rng.random() < 0.6, cache=cache, packed=packed, single=rng.choice([0.0, 0.7]), pick=pick)


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _case(name, **rest):
    return rest if name is None else dict(name=name, **rest)


def _rotary(name, windows, tokens, heads, head_dim, part, layout, far, dtype='bf16', gradient=False, stretch=1.0,
            amplitude=1.0):
    return _case(name, kind='rotary', windows=windows, tokens=tokens, heads=heads, head_dim=head_dim, part=part,
                 layout=layout, far=far, dtype=dtype, gradient=gradient, stretch=stretch, amplitude=amplitude)


def _append(name, windows, low, high, held, heads, head_dim, page, turn, cache='bf16', packed=False, pick=3):
    return _case(name, kind='append', windows=windows, low=low, high=high, held=held, heads=heads, head_dim=head_dim,
                 page=page, turn=turn, cache=cache, packed=packed, pick=pick)


def _attend(name, windows, low, high, short, long, heads, groups, head_dim, page, causal=False, cache='bf16',
            packed=False, single=0.0, pick=5):
    return _case(name, kind='attend', windows=windows, low=low, high=high, short=short, long=long, heads=heads,
                 groups=groups, head_dim=head_dim, page=page, causal=causal, cache=cache, packed=packed, single=single,
                 pick=pick)


def _counts(case):
    """Each window's new tokens; one has the most."""
    rng = random.Random(case['pick'])
    n = [1 if rng.random() < case.get('single', 0.0) else rng.randint(case['low'], case['high'])
         for _ in range(case['windows'])] if case['packed'] else [case['high']] * case['windows']
    n[rng.randrange(len(n))] = case['high']
    return n


def _lengths(case):
    """Each window's keys, the new tokens' among them; one has the most."""
    rng = random.Random(case['pick'] + 1)
    if case['kind'] == 'append':
        return [rng.randint(case['held'] // 2, case['held']) + n for n in _counts(case)]
    L = [rng.randint(case['short'], case['long']) for _ in range(case['windows'])]
    L[rng.randrange(len(L))] = case['long']
    return L


# -------------------------------------------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(DEVICE).manual_seed(seed)


def _normal(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEVICE, generator=g).to(dtype)


def _frequencies(part, stretch):
    return (10000.0 ** (-torch.arange(0, part, 2, dtype=torch.float64) / part) / stretch).to(DEVICE)


def _codes(x):
    """Normal values as e4m3 codes of rows whose exponent is 120 (2^-7)."""
    return (x.float() * 128).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _pool(case, g, lengths):
    """A pool of pages in use and spare ones, the windows' pages scattered over it, filled with earlier values."""
    H = case['heads'] // case.get('groups', 1)
    S, D = case['page'], case['head_dim']
    need = [-(-L // S) for L in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, device=DEVICE, generator=g).to(torch.int32)
    table = torch.zeros(len(need), max(max(need), 1), dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    k, v = _normal(g, pages, H, S, D), _normal(g, pages, H, S, D)
    lengths = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    pool = dict(k=k, v=v, table=table, lengths=lengths, ke=None, ve=None)
    if case['cache'] == 'fp8':
        pool['k'], pool['v'] = _codes(k), _codes(v)
        pool['ke'] = torch.randint(119, 122, (pages, H, S), device=DEVICE, generator=g).to(torch.uint8)
        pool['ve'] = torch.randint(119, 122, (pages, H, S), device=DEVICE, generator=g).to(torch.uint8)
    return pool


def prepare(case, seed):
    g = _generator(seed)
    kind, D = case['kind'], case['head_dim']
    if kind == 'rotary':
        B, N, H = case['windows'], case['tokens'], case['heads']
        dtype = torch.float32 if case['dtype'] == 'fp32' else torch.bfloat16
        x = _normal(g, B, N, H, D, dtype=dtype).transpose(1, 2)      # a projection's rows, heads before tokens
        first = torch.randint(max(1, case['far'] - N + 1), (B, 1), device=DEVICE, generator=g)
        positions = first + torch.arange(N, device=DEVICE)
        state = dict(case=case, x=x, positions=positions, frequencies=_frequencies(case['part'], case['stretch']))
        if case['gradient']:
            state['x'] = x.requires_grad_()
            state['dy'] = _normal(g, B, N, H, D, dtype=dtype).transpose(1, 2)
        return state
    counts, lengths = _counts(case), _lengths(case)
    state = dict(case=case, most=max(counts), longest=max(lengths), **_pool(case, g, lengths))
    T, B = sum(counts), len(counts)
    state['cu'] = None
    if case['packed']:
        state['cu'] = torch.tensor([0] + counts, device=DEVICE).cumsum(0).to(torch.int32)
    if kind == 'append':
        H = case['heads']
        rows = _normal(g, T, 2, H, D)                                 # the key / value projection of the new tokens
        heads_first = (lambda t: t.transpose(0, 1)) if case['packed'] else (
            lambda t: t.view(B, case['high'], H, D).transpose(1, 2))
        kv = [rows[:, 0], rows[:, 1]]
        state['key'], state['value'] = [heads_first(t) if case['packed'] else heads_first(t.contiguous()) for t in kv]
        state['positions'] = state['frequencies'] = None
        if case['turn'] == 'axial':
            state['positions'] = torch.rand(T, 3, device=DEVICE, generator=g) * 64 - 8
            if not case['packed']:
                state['positions'] = state['positions'].view(B, case['high'], 3)
            axis = D // 3
            state['frequencies'] = (10000.0 ** (-torch.arange(0, axis, 2).float() / axis)).to(DEVICE)
        elif case['turn'] != 'none':
            state['frequencies'] = _frequencies(D, 1.0)
        return state
    H = case['heads']
    rows = 1.5 * _normal(g, T, H, D)
    state['query'] = rows.transpose(0, 1) if case['packed'] else rows.view(B, case['high'], H, D).transpose(1, 2)
    return state


# ------------------------------------------------------------------------------------------------ the measured calls

def run(state):
    case = state['case']
    if own:
        return _own(state, case)
    if case['kind'] == 'rotary':
        if not case['gradient']:
            return _plain_rotary(state['x'], state, case, 1.0)
        x, dy = state['x'].detach(), state['dy']
        return _plain_rotary(x, state, case, 1.0), _plain_rotary(dy, state, case, -1.0)
    if case['kind'] == 'append':
        return _plain_append(state, case)
    return _plain_attend(state, case)


def _own(state, case):
    from streamvoxel_amd.stream.paged import paged_append, paged_attention
    from streamvoxel_amd.stream.rotary import rotary
    if case['kind'] == 'rotary':
        y = rotary(state['x'], state['positions'], state['frequencies'], layout=case['layout'],
                   amplitude=case['amplitude'])
        if not case['gradient']:
            return y
        return y.detach(), torch.autograd.grad(y, state['x'], state['dy'])[0]
    if case['kind'] == 'append':
        paged_append(state['key'], state['value'], state['k'], state['v'], state['table'], state['lengths'],
                     cu_tokens=state['cu'], positions=state['positions'], frequencies=state['frequencies'],
                     layout=case['turn'] if case['turn'] != 'none' else 'half', k_exponents=state['ke'],
                     v_exponents=state['ve'])
        return _written(state)
    return paged_attention(state['query'], state['k'], state['v'], state['table'], state['lengths'],
                           cu_queries=state['cu'], causal=case['causal'], k_exponents=state['ke'],
                           v_exponents=state['ve'])


def _written(state):
    if state['ke'] is None:
        return state['k'], state['v']
    return state['k'], state['v'], state['ke'], state['ve']


def _turned(x, cos, sin, layout):
    """The pairs of x [..., part] turned by cos / sin [..., part / 2]."""
    if layout == 'half':
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _plain_rotary(x, state, case, sign):
    angle = state['positions'].double()[..., None] * state['frequencies']          # [B, N, part / 2]
    cos = (case['amplitude'] * angle.cos()).float()[:, None]
    sin = (sign * case['amplitude'] * angle.sin()).float()[:, None]
    part = case['part']
    turned = _turned(x[..., :part].float(), cos, sin, case['layout'])
    return torch.cat((turned, x[..., part:].float()), -1).to(x.dtype)


def _tokens(state, case, rows):
    """(window, key index) of every new token, windows one after the other."""
    lengths = state['lengths'].long()
    if case['packed']:
        cu = state['cu'].long()
        t = torch.arange(rows, device=DEVICE)
        b = torch.searchsorted(cu[1:], t, right=True)
        return b, lengths[b] - cu[b + 1] + t
    n = state['most']
    b = torch.arange(case['windows'], device=DEVICE).repeat_interleave(n)
    return b, lengths[b] - n + torch.arange(n, device=DEVICE).repeat(case['windows'])


def _row_codes(x, bound):
    """Rows x [T, H, D] as e4m3 codes under the least power of two that holds bound [T, H], and its exponent."""
    mantissa, exponent = torch.frexp(bound)
    code = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8) + 127
    code = torch.where(bound == 0, torch.ones_like(code), code).clamp(1, 254)
    return (x * _power(254 - code)[..., None]).to(torch.float8_e4m3fn), code.to(torch.uint8)


def _power(code):
    """2^(code - 127) in fp32, by its bits."""
    return (code.int() << 23).view(torch.float32)


def _plain_append(state, case):
    flat = (lambda t: t.transpose(0, 1)) if case['packed'] else (lambda t: t.transpose(1, 2).flatten(0, 1))
    key, value = flat(state['key']).float(), flat(state['value']).float()           # [T, H, D]
    b, at = _tokens(state, case, len(key))
    page, row = state['table'].long()[b, at // case['page']], at % case['page']
    turned, reach = key, 1.0
    if case['turn'] == 'axial':
        turned, reach = _plain_axial(key, state['positions'].reshape(-1, 3), state['frequencies']), 1.5
    elif case['turn'] != 'none':
        angle = at.double()[:, None] * state['frequencies']
        turned = _turned(key, angle.cos().float()[:, None], angle.sin().float()[:, None], case['turn'])
        reach = 1.5
    if state['ke'] is None:
        state['k'][page, :, row] = turned.to(torch.bfloat16)
        state['v'][page, :, row] = value.to(torch.bfloat16)
        return _written(state)
    codes, state['ke'][page, :, row] = _row_codes(turned, reach * key.abs().amax(-1))
    state['k'].view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
    codes, state['ve'][page, :, row] = _row_codes(value, value.abs().amax(-1))
    state['v'].view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
    return _written(state)


def _plain_axial(key, positions, frequencies):
    """The three-axis rotation as the framework defines it on bf16 activations: a phase of one fp32 product, sin, cos,
    every product and every sum rounded to bf16."""
    low = lambda t: t.to(torch.bfloat16).float()
    phase = positions[:, :, None] * frequencies                                     # [T, 3, D / 6]
    cos, sin = low(phase.double().cos().float()), low(phase.double().sin().float())
    cos, sin = cos.flatten(1)[:, None], sin.flatten(1)[:, None]
    a, b = key[..., 0::2], key[..., 1::2]
    return torch.stack((low(low(a * cos) - low(b * sin)), low(low(a * sin) + low(b * cos))), -1).flatten(-2)


def _held(pages, exponents, table, count):
    """Keys or values of every window [B, H, count, D] in fp32."""
    S = pages.shape[2]
    table = table[:, :-(-count // S)].long()
    x = pages.view(torch.uint8)[table].view(pages.dtype).float() if exponents is not None else pages[table].float()
    if exponents is not None:
        x = x * _power(exponents[table])[..., None]
    return x.transpose(1, 2).flatten(2, 3)[:, :, :count]


def _plain_attend(state, case):
    B, H, D, n, G = case['windows'], case['heads'], case['head_dim'], state['most'], case['groups']
    lengths = state['lengths'].long()
    query = state['query']
    counts = torch.full((B,), n, device=DEVICE)
    if case['packed']:
        b, at = _tokens(state, case, query.shape[1])
        counts = (state['cu'][1:] - state['cu'][:-1]).long()
        i = at - lengths[b] + counts[b]
        padded = torch.zeros(B, n, H, D, device=DEVICE)
        padded[b, i] = query.transpose(0, 1).float()
        query = padded.transpose(1, 2)
    k = _held(state['k'], state['ke'], state['table'], state['longest'])            # [B, H / G, L, D]
    v = _held(state['v'], state['ve'], state['table'], state['longest'])
    q = query.float().reshape(B, H // G, G * n, D)                                  # a key head's heads and tokens
    scores = q @ k.transpose(2, 3) / math.sqrt(D)
    j = torch.arange(state['longest'], device=DEVICE)
    last = lengths[:, None] - 1
    if case['causal']:
        last = lengths[:, None] - counts[:, None] + torch.arange(n, device=DEVICE)
    last = last.expand(B, n).repeat(1, G)                                           # [B, G n]
    scores = scores.masked_fill(j > last[:, None, :, None], -math.inf)
    weight = (scores - scores.amax(-1, keepdim=True).clamp(min=-3e38)).exp()
    total = weight.sum(-1, keepdim=True)
    out = (weight @ v) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.reshape(B, H, n, D)
    if case['packed']:
        out = out.transpose(1, 2)[b, i].transpose(0, 1)
    return out.to(torch.bfloat16)


# --------------------------------------------------------------------------------------------------- what it takes

def work(case):
    kind, H, D = case['kind'], case['heads'], case['head_dim']
    if kind == 'rotary':
        rows, passes = case['windows'] * case['tokens'], 2 if case['gradient'] else 1
        wide = 4 if case['dtype'] == 'fp32' else 2
        return dict(bytes=passes * 2 * wide * rows * H * D + 8 * rows + 4 * case['part'],
                    flops=passes * 3 * rows * H * case['part'])
    counts, lengths = _counts(case), _lengths(case)
    if kind == 'append':
        rows = sum(counts) * H
        turn = 0 if case['turn'] == 'none' else 3
        held = 2 * (D + 1) if case['cache'] == 'fp8' else 4 * D
        return dict(bytes=rows * (4 * D + held) + 4 * sum(-(-L // case['page']) for L in lengths),
                    flops=turn * rows * D)
    row = D + 1 if case['cache'] == 'fp8' else 2 * D
    keys, pairs = sum(lengths), 0
    for n, L in zip(counts, lengths):
        pairs += n * L - (n * (n - 1) // 2 if case['causal'] else 0)
    return dict(bytes=4 * sum(counts) * H * D + 2 * keys * (H // case['groups']) * row
                + 4 * sum(-(-L // case['page']) for L in lengths), flops=4 * H * D * pairs)


# ------------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    kind, D = case['kind'], case['head_dim']
    if kind == 'rotary':
        def rotated(x, sign):
            y, half = x.detach().double().clone(), case['part'] // 2
            for i in range(half):
                a, b = (i, i + half) if case['layout'] == 'half' else (2 * i, 2 * i + 1)
                angle = state['positions'].double() * float(state['frequencies'][i])
                c, s = case['amplitude'] * angle.cos()[:, None], sign * case['amplitude'] * angle.sin()[:, None]
                xa, xb = x.detach()[..., a].double(), x.detach()[..., b].double()
                y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
            return y
        return (rotated(state['x'], 1.0), rotated(state['dy'], -1.0)) if case['gradient'] else rotated(state['x'], 1.0)
    counts, lengths, S = _counts(case), _lengths(case), case['page']
    if kind == 'append':
        # The exponents are whole numbers; the three-axis rotation is defined by its roundings and has no such value.
        fp8, axial = case['cache'] == 'fp8', case['turn'] == 'axial'
        k, v = state['k'].float().double(), state['v'].float().double()
        at = 0
        for b, (n, L) in enumerate(zip(counts, lengths)):
            cut = (lambda t: t[:, at:at + n]) if case['packed'] else (lambda t: t[b])
            key, value = cut(state['key']).double(), cut(state['value']).double()   # [H, n, D]
            bounds = key.abs().amax(-1) * (1.0 if case['turn'] == 'none' else 1.5), value.abs().amax(-1)
            where = torch.arange(L - n, L, device=DEVICE)
            if case['turn'] in ('half', 'interleaved'):
                z = where.double()[:, None] * state['frequencies']
                spin = torch.polar(torch.ones_like(z), z)
                pair = key.unflatten(-1, (2, D // 2)).transpose(-1, -2) if case['turn'] == 'half' else (
                    key.unflatten(-1, (D // 2, 2)))
                pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * spin)
                key = (pair.transpose(-1, -2) if case['turn'] == 'half' else pair).flatten(-2)
            if fp8:
                key, value = [x / 2.0 ** torch.ceil(torch.log2(most / E4M3_MAX))[..., None]
                              for x, most in zip((key, value), bounds)]
            page = state['table'][b].long()[where // S]
            k[page, :, where % S], v[page, :, where % S] = key.transpose(0, 1), value.transpose(0, 1)
            at += n
        return (None if axial else k, v) + ((None, None) if fp8 else ())
    if work(case)['flops'] > 4e12:
        return None
    G, outs, at = case['groups'], [], 0
    for b, (n, L) in enumerate(zip(counts, lengths)):
        q = (state['query'][:, at:at + n] if case['packed'] else state['query'][b]).double()      # [H, n, D]
        at += n
        page = state['table'][b, :-(-L // S)].long()
        rows = []
        for pages, exponents in ((state['k'], state['ke']), (state['v'], state['ve'])):
            x = pages.view(torch.uint8)[page].view(pages.dtype) if exponents is not None else pages[page]
            x = x.float().double()
            if exponents is not None:
                x = x * 2.0 ** (exponents[page].double() - 127)[..., None]
            rows.append(x.transpose(0, 1).reshape(x.shape[1], -1, D)[:, :L])
        out = torch.empty_like(q)
        for h in range(case['heads']):
            z = q[h] @ rows[0][h // G].t().contiguous() * D ** -0.5
            if case['causal']:
                seen = torch.ones(n, L, dtype=torch.bool, device=DEVICE).tril(L - n)
                z = torch.where(seen, z, torch.full_like(z, -math.inf))
            out[h] = torch.softmax(z, -1) @ rows[1][h // G]
        outs.append(out)
    return torch.cat(outs, 1) if case['packed'] else torch.stack(outs)
