"""A paged cache of keys and values on the HIP kernels: the append that fills it, the attention over it, and the context
that stands in `CachedContext`'s place with its windows in one pool of pages.

`step.CachedContext` (PackedKeys, streamvoxel/stream/fast_ops.py:122-159) keeps a slab of the longest condition for
every slot and rewrites it whole; here a window holds the pages that its keys fill, and new keys go behind the ones
that are there. No counterpart in the reference.
"""
from __future__ import annotations

import struct

import torch

from streamvoxel_amd import _lib

__all__ = ['paged_append', 'paged_attention', 'PagedContext']

LAYOUTS = {'half': _lib.SVHIP_ROTARY_HALF, 'interleaved': _lib.SVHIP_ROTARY_INTERLEAVED,
           'axial': _lib.SVHIP_ROTARY_AXIAL}


def _check_pool(k_pages, v_pages, page_table, lengths, k_exponents, v_exponents, bad):
    """The pool's type code; ValueError / TypeError for what the kernels do not take."""
    shape, dtype = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype != dtype:
        raise ValueError('k_pages and v_pages must be [pages, heads, page, head_dim] alike')
    if k_pages.stride(-1) != 1 or v_pages.stride(-1) != 1:
        raise ValueError('rows of a page need a contiguous head_dim')
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError('page_table must be int32 [B, pages of a window] with contiguous rows')
    if lengths.dtype != torch.int32 or lengths.shape != page_table.shape[:1] or not lengths.is_contiguous():
        raise ValueError('lengths must be a contiguous int32 [B]')
    if bad is not None and (bad.dtype != torch.int32 or bad.numel() != 1):
        raise ValueError('bad must be one int32')
    if dtype == torch.bfloat16:
        if k_exponents is not None or v_exponents is not None:
            raise TypeError('bf16 pages take no exponents')
        return _lib.SVHIP_BF16
    if dtype != torch.float8_e4m3fn:
        raise TypeError(f'pages of {dtype} unsupported (bfloat16 or float8_e4m3fn)')
    for e in (k_exponents, v_exponents):
        if e is None or e.dtype != torch.uint8 or e.shape != shape[:3] or e.stride(-1) != 1:
            raise ValueError('e4m3 pages need k_exponents and v_exponents, uint8 [pages, heads, page] with contiguous '
                             'rows')
    return _lib.SVHIP_FP8_E4M3


def _windows(t, cu, B, what):
    """(heads, tokens, (stride of a window, of a head, of a token)) of [B,H,n,D], or packed [H,T,D] with borders cu."""
    shape, stride = t.shape, t.stride()
    if cu is None:
        if len(shape) != 4 or shape[0] != B:
            raise ValueError(f'{what} must be [B, heads, n, head_dim] with the B windows of the table, or packed '
                             '[heads, T, head_dim] with their borders')
        return shape[1], shape[2], stride[:3]
    if cu.dtype != torch.int32 or cu.shape != (B + 1,) or not cu.is_contiguous():
        raise ValueError('the borders must be a contiguous int32 [B + 1]')
    if len(shape) != 3:
        raise ValueError(f'packed {what} must be [heads, T, head_dim]')
    return shape[0], shape[1], (0, *stride[:2])


def _rows16(t):
    """bf16 rows on 16-byte boundaries: the tensor itself, or a contiguous copy."""
    *rows, last = t.stride()
    off = t.data_ptr() >> 1
    for s in rows:
        off |= s
    if last == 1 and off & 7 == 0:
        return t
    # (The stride of a dimension with one element is never used, and may be anything.)
    if last == 1 and (t.data_ptr() >> 1) & 7 == 0 and all(s & 7 == 0 for n, s in zip(t.shape, rows) if n > 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


_CACHE = struct.Struct('7P18q')    # svhip_paged_cache
_APPEND = struct.Struct('5P13qd')  # svhip_paged_append_args
_ATTEND = struct.Struct('4P10qd')  # svhip_paged_attention_args


def _address(t):
    return 0 if t is None else t.data_ptr()


def _packed(code, k_pages, v_pages, page_table, lengths, k_exponents, v_exponents, bad):
    """The svhip_paged_cache of checked tensors."""
    P, H, S, D = k_pages.shape
    ke, ve = (0, 0), (0, 0)
    if k_exponents is not None:
        ke, ve = k_exponents.stride()[:2], v_exponents.stride()[:2]
    return _CACHE.pack(k_pages.data_ptr(), v_pages.data_ptr(), _address(k_exponents), _address(v_exponents),
                       page_table.data_ptr(), lengths.data_ptr(), _address(bad), code, page_table.shape[0], H, D, P, S,
                       page_table.shape[1], page_table.stride(0), *k_pages.stride()[:3], *v_pages.stride()[:3], *ke, *ve)


def paged_append(key, value, k_pages, v_pages, page_table, lengths, cu_tokens=None, before=0, positions=None,
                 frequencies=None, layout='half', amplitude=1.0, k_exponents=None, v_exponents=None, bad=None):
    """The windows' new keys and values into their rows of a paged cache, the keys rotated on the way.

    key, value bf16 [B,H,n,D] (head_dim contiguous, any other strides), or packed [H,T,D] with the windows' borders
    `cu_tokens` int32 [B+1] (device, ascending; tokens outside every window are left alone). k_pages, v_pages
    [pages,H,page,D] in bf16, or float8_e4m3fn with `k_exponents` / `v_exponents` uint8 [pages,H,page], one power of
    two 2^(exponent - 127) for each row (written too, 1 to 254); page a power of two from 16 to 1024. page_table int32 [B, m]:
    key j of window b is row j % page of page page_table[b, j // page]. `lengths` int32 [B] (device) counts each
    window's keys with the new ones: they are its last n keys, or the n in front of its last `before`. Two tokens must
    not share a row. `frequencies` rotates the keys: with layout 'half' / 'interleaved' as `rotary` does (fp64;
    `positions` int32 / int64 [B,n] or [T], or None: each key's index in its window; `amplitude`), with 'axial' as
    `producer.axial_rope` does (its fp32 buffer and fp32 positions [B,n,3] or [T,3]). `bad` (optional int32 [1],
    device) becomes 1 when a key lies outside its window's row of the table or a page outside the pool; such keys are
    not written."""
    _lib.require_one_gpu(key, value, k_pages, v_pages, page_table, lengths, cu_tokens, positions, frequencies, k_exponents,
                         v_exponents, bad)
    code = _check_pool(k_pages, v_pages, page_table, lengths, k_exponents, v_exponents, bad)
    if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
        raise TypeError('key and value must be bfloat16')
    key, value = _rows16(key), _rows16(value)
    B = page_table.shape[0]
    H, n, sk = _windows(key, cu_tokens, B, 'key')
    sv = _windows(value, cu_tokens, B, 'value')[2]
    P, Hp, S, D = k_pages.shape
    if value.shape != key.shape or H != Hp or key.shape[-1] != D:
        raise ValueError('key and value must be alike, with the heads and the head_dim of the pages')
    if before < 0:
        raise ValueError('before counts keys')
    for k, v in ((k_pages, v_pages), (k_exponents, v_exponents)):
        if k is None:
            break
        if _lib.stacked(k) or _lib.stacked(v):
            raise ValueError('pages and their exponents must have a place for every element')
        if k.data_ptr() == v.data_ptr() and k.numel():
            raise ValueError('keys and values must not share their pages or exponents')
    wide, pairs, sp, turn = 0, 0, (0, 0), _lib.SVHIP_ROTARY_NONE
    if frequencies is not None:
        if layout not in LAYOUTS:
            raise ValueError("layout is 'half', 'interleaved' or 'axial'")
        turn, tokens = LAYOUTS[layout], (n,) if cu_tokens is not None else (B, n)
        if layout == 'axial':
            if frequencies.dtype != torch.float32 or frequencies.numel() * 6 != D or not frequencies.is_contiguous():
                raise ValueError('frequencies must be the fp32 [head_dim / 6] buffer')
            if positions is None or positions.dtype != torch.float32 or tuple(positions.shape) != (*tokens, 3) or (
                    positions.stride(-1) != 1):
                raise ValueError("the 'axial' layout needs fp32 positions, three a token")
            pairs = D // 2
        else:
            if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous():
                raise ValueError('frequencies must be a contiguous fp64 vector')
            pairs = frequencies.numel()
            if not 1 <= pairs <= D // 2:
                raise ValueError(f'{pairs} frequencies do not fit head_dim {D}')
            if positions is not None and (positions.dtype not in (torch.int32, torch.int64)
                                          or tuple(positions.shape) != tokens):
                raise ValueError('positions must be int32 or int64, one a token')
        if positions is not None:
            wide = int(positions.dtype == torch.int64)
            sp = (0, positions.stride(0)) if cu_tokens is not None else (positions.stride(0), positions.stride(1))
    elif positions is not None:
        raise ValueError('rotating the keys needs frequencies')
    args = _APPEND.pack(key.data_ptr(), value.data_ptr(), _address(cu_tokens), _address(positions), _address(frequencies),
                        n, before, *sk, *sv, turn, wide, *sp, pairs, amplitude)
    cache = _packed(code, k_pages, v_pages, page_table, lengths, k_exponents, v_exponents, bad)
    _lib.launch('svhip_paged_append', key, cache, args)


def paged_attention(query, k_pages, v_pages, page_table, lengths, cu_queries=None, causal=False, scale=None,
                    k_exponents=None, v_exponents=None, out=None, bad=None):
    """softmax(scale * Q K^T) V of the windows' new tokens over the first lengths[b] keys of their pages.

    query bf16 [B,H,n,D] (head_dim contiguous, any other strides), or packed [H,T,D] with the windows' borders
    `cu_queries` int32 [B+1] (device, ascending). k_pages, v_pages, page_table, lengths and the exponents as
    `paged_append` fills them; the H heads share the pages' heads evenly, head h reads head h // (H / heads).
    `causal`: the n tokens are the window's last n keys, and token i sees keys up to its own, lengths[b] - n + i;
    without it every token sees all of them. A token with no key gets zeros, and what is not finite among keys that a
    token does not see does not reach it. The same call gives the same bits; other windows in the call move the places
    where a window's keys are cut for several workgroups, and with them its last bits (`attention` keeps a window's bits
    in any batch). `out` (optional; query itself, or memory that query does not share) bf16
    like query with a contiguous head_dim; its rows outside every window are left as they are (a fresh one has them
    undefined). `bad` (optional int32 [1], device) becomes 1 when a page lies outside the pool (its keys and values
    read as zeros) or a length passes the window's row of the table (and is cut). Takes no part in a gradient. Returns
    out."""
    _lib.require_one_gpu(query, k_pages, v_pages, page_table, lengths, cu_queries, k_exponents, v_exponents, out, bad)
    code = _check_pool(k_pages, v_pages, page_table, lengths, k_exponents, v_exponents, bad)
    if query.dtype != torch.bfloat16:
        raise TypeError('query must be bfloat16')
    given, query = query, _rows16(query)
    B = page_table.shape[0]
    H, n, sq = _windows(query, cu_queries, B, 'query')
    P, Hkv, S, D = k_pages.shape
    if query.shape[-1] != D or Hkv == 0 or H % Hkv:
        raise ValueError("query needs the pages' head_dim, and heads that share theirs evenly")
    if out is None:
        out = torch.empty_like(query)
    elif out.shape != query.shape or out.dtype != torch.bfloat16 or out.stride(-1) != 1 or _lib.stacked(out):
        raise ValueError('out must be bf16 like query with a contiguous head_dim and a place for every element')
    elif _lib.overlaps(given, out) and (given.data_ptr() != out.data_ptr() or given.stride() != out.stride()):
        raise ValueError('out must be query itself or memory that query does not share')
    so = _windows(out, cu_queries, B, 'out')[2]
    scale = D ** -0.5 if scale is None else float(scale)
    nbytes = _lib.load().svhip_paged_attention_workspace_bytes(B, H, Hkv, n, cu_queries is not None, D,
                                                               page_table.shape[1] * S)
    cache = _packed(code, k_pages, v_pages, page_table, lengths, k_exponents, v_exponents, bad)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=query.device) if nbytes else None
    args = _ATTEND.pack(query.data_ptr(), out.data_ptr(), _address(cu_queries), _address(ws), nbytes, H, n, *sq, *so, causal,
                        scale)
    _lib.launch('svhip_paged_attention', query, cache, args)
    return out


class PagedContext:
    """The cached keys and values of `batch` windows in one pool of `pages` pages a layer (each `page_size` keys of
    every head), in `CachedContext`'s place: `write`, `attend`, `lengths` as there, and windows that grow (`grow`,
    `append`) and give their pages back (`release`). A window holds as many pages as its keys need, at most
    `max_pages` of them (default: all). kv_dtype 'bf16' or 'fp8' (OCP e4m3fn with one power of two for each row and
    head).

    What it costs beside the slab: the attention of 1024 queries a window takes 6 to 14 % longer at head_dim 64 (a tenth
    to a fifth less at 128), and a window's last bits depend on the other windows of the call (`paged_attention`), where
    `CachedContext` gives a window the same bits in any batch.

    The host keeps the books: `resize` and `grow` take and free pages and send the window's table and length to the
    device on the current stream without waiting for it; calls that touch a window's pages must be ordered after them,
    as usual. Other windows may be in work on other streams: a page that changes hands is waited for. A replayed graph
    reads the table and the lengths as they stand; a capture that would change them is refused. `bad` (device int32
    [1]) becomes non-zero when a call meets a page outside the pool, which these books never name."""

    def __init__(self, layers, batch, heads, head_dim, pages, device, page_size=64, max_pages=None, kv_dtype='bf16'):
        if kv_dtype not in ('bf16', 'fp8'):
            raise ValueError("kv_dtype must be 'bf16' or 'fp8'")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError('page_size must be a power of two from 16 to 1024')
        if head_dim < 8 or head_dim > 128 or head_dim % 8:
            raise ValueError('head_dim must be a multiple of 8 up to 128')
        if layers < 1 or batch < 1 or heads < 1 or pages < 1 or (max_pages is not None and max_pages < 1):
            raise ValueError('layers, batch, heads, pages and max_pages must be positive')
        self.layers, self.batch, self.heads, self.head_dim = layers, batch, heads, head_dim
        self.pages, self.page_size, self.kv_dtype = pages, page_size, kv_dtype
        self.max_pages = pages if max_pages is None else max_pages
        dt = torch.bfloat16 if kv_dtype == 'bf16' else torch.float8_e4m3fn
        pool = lambda dtype, *shape: [torch.empty(pages, heads, page_size, *shape, dtype=dtype, device=device)
                                      for _ in range(layers)]
        self.k, self.v = pool(dt, head_dim), pool(dt, head_dim)
        none = [None] * layers
        self.k_exponents, self.v_exponents = (pool(torch.uint8), pool(torch.uint8)) if kv_dtype == 'fp8' else (none, none)
        self.table = torch.zeros(batch, self.max_pages, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.bad = torch.zeros(1, dtype=torch.int32, device=device)
        self.host_lengths = [0] * batch
        self._owned = [[] for _ in range(batch)]
        self._free = list(range(pages - 1, -1, -1))
        self._left = {}        # free page -> (stream that it was given back on, event there)

    @property
    def free_pages(self):
        return len(self._free)

    def _stream(self):
        return torch.cuda.current_stream(self.lengths.device) if self.lengths.is_cuda else None

    def _capturing(self):
        return self.lengths.is_cuda and torch.cuda.is_current_stream_capturing()

    def _pages_for(self, length):
        return -(-length // self.page_size)

    def _set(self, wanted):
        """The windows' lengths {index: length}: pages taken and freed, table and lengths sent. Nothing changes on
        error."""
        self._take(wanted)
        changed = sorted(index for index, length in wanted.items() if length != self.host_lengths[index])
        for index in changed:
            self.host_lengths[index] = wanted[index]
        self._send_lengths(changed)

    def _take(self, wanted):
        """Pages for the windows' lengths {index: length} taken and freed, and the table sent."""
        need = 0
        for index, length in wanted.items():
            if not 0 <= index < self.batch:
                raise IndexError(f'window {index} of {self.batch}')
            if length < 0:
                raise ValueError('a window holds 0 keys or more')
            if self._pages_for(length) > self.max_pages:
                raise ValueError('Condition exceeds the slot capacity')
            need += self._pages_for(length) - len(self._owned[index])
        if need > len(self._free):
            raise RuntimeError(f'the pool has {len(self._free)} pages left, {need} more are needed')
        stream, freed, moved = self._stream(), [], []
        if self._capturing():
            raise RuntimeError('the books of a PagedContext are kept by the host: change them outside the capture')
        for index, length in wanted.items():          # freed pages first: another window may take them
            own, n = self._owned[index], self._pages_for(length)
            if n != len(own):
                moved.append(index)
            freed.extend(reversed(own[n:]))
            del own[n:]
        self._free.extend(freed)
        if freed and stream is not None:
            self._left.update(dict.fromkeys(freed, (stream, stream.record_event())))
        taken = []
        for index, length in wanted.items():
            own, n = self._owned[index], self._pages_for(length)
            new = [self._free.pop() for _ in range(n - len(own))]
            own.extend(new)
            taken.extend(new)
        # A page given back on another stream may still be in work there.
        for left, event in {self._left.pop(page) for page in taken if page in self._left}:
            if left != stream:
                stream.wait_event(event)
        for index in moved:
            self._send(self.table[index, :len(self._owned[index])], self._owned[index])

    def _send_lengths(self, windows):
        """The lengths of these windows (ascending) alone: a call for another window may be on its way on another
        stream."""
        runs = []
        for index in windows:
            if runs and runs[-1][1] == index:
                runs[-1][1] = index + 1
            else:
                runs.append([index, index + 1])
        if len(runs) > 2:          # in one copy
            both = torch.empty(2, len(windows), dtype=torch.int32, device=self.lengths.device)
            self._send(both.view(-1), windows + [self.host_lengths[index] for index in windows])
            self.lengths.index_copy_(0, both[0].long(), both[1])
            return
        for first, end in runs:
            self._send(self.lengths[first:end], self.host_lengths[first:end])

    @staticmethod
    def _send(to, values):
        """Host numbers to the device on the current stream, not waited for: one by a fill, more from pinned memory
        (which the allocator keeps until the copy is done)."""
        if len(values) == 1:
            to.fill_(values[0])
        elif values:
            to.copy_(torch.tensor(values, dtype=torch.int32, pin_memory=True), non_blocking=True)

    def resize(self, index, length):
        """Window `index` holds `length` keys: pages taken or given back at its end (the keys below both lengths
        stay)."""
        self._set({int(index): int(length)})

    def reserve(self, index, length):
        """Window `index` takes the pages of `length` keys, at least as many as it holds, and holds no more for now:
        `append` with `lengths` writes the new ones, `resize` then makes them seen."""
        if 0 <= index < self.batch and length < self.host_lengths[index]:
            raise ValueError(f'window {index} holds {self.host_lengths[index]} keys')
        self._take({int(index): int(length)})

    def release(self, index):
        """Window `index` gives its pages back."""
        self.resize(index, 0)

    def grow(self, counts):
        """Every window grows by counts[b] keys (or all by one number), to be written by `append`."""
        counts = [int(counts)] * self.batch if isinstance(counts, int) else [int(c) for c in counts]
        if len(counts) != self.batch or min(counts) < 0:
            raise ValueError(f'counts must be {self.batch} numbers, 0 or more')
        self._set({b: self.host_lengths[b] + c for b, c in enumerate(counts)})

    def _rows(self, t):
        t = t.to(device=self.lengths.device, dtype=torch.bfloat16)
        return t if t.stride(-1) == 1 else t.contiguous()

    def append(self, layer, key, value, index=None, n=None, cu_tokens=None, lengths=None, **how):
        """`paged_append` into layer `layer` of the first n windows (all by default), or of window `index` alone (key,
        value [heads, L, head_dim] then); `lengths` (default: the windows') counts the keys with the new ones; `how`:
        its before, positions, frequencies, layout, amplitude."""
        at = slice(0, self.batch if n is None else n)
        if index is not None:
            at, key, value = slice(index, index + 1), key[None], value[None]
            if how.get('positions') is not None:
                how['positions'] = how['positions'][None]
        lengths = self.lengths[at] if lengths is None else lengths
        paged_append(key, value, self.k[layer], self.v[layer], self.table[at], lengths, cu_tokens=cu_tokens,
                     k_exponents=self.k_exponents[layer], v_exponents=self.v_exponents[layer], bad=self.bad, **how)

    def write(self, layer, index, key, value, prefix=None, positions=None, frequencies=None):
        """Window `index` of `layer` anew, as `CachedContext.write`: keys [0, P) from `prefix` = (prefix_k, prefix_v)
        [H, P, D] (already rotated), keys [P, P + L) from key, value [H, L, D] (K rotated by AxialRoPE at fp32
        positions [L, 3] with the fp32 `frequencies` buffer when given). Sets the window's length and pages."""
        _lib.require_gpu(key, value)
        key, value = self._rows(key), self._rows(value)
        H, L, D = key.shape
        if H != self.heads or D != self.head_dim or value.shape != key.shape:
            raise ValueError('key / value must be [heads, L, head_dim] like the cache')
        P = 0
        if prefix is not None:
            pk, pv = self._rows(prefix[0]), self._rows(prefix[1])
            if pk.shape[0] != H or pk.shape[2] != D or pv.shape != pk.shape:
                raise ValueError('prefix K / V must be [heads, P, head_dim]')
            P = pk.shape[1]
        how = {}
        if positions is not None:
            if frequencies is None:
                raise ValueError('rotating the local keys needs the AxialRoPE frequencies')
            dev = self.lengths.device
            how = dict(positions=positions.to(device=dev, dtype=torch.float32).contiguous(), layout='axial',
                       frequencies=frequencies.to(device=dev, dtype=torch.float32).contiguous())
            if how['positions'].shape != (L, 3):
                raise ValueError('positions must be [L, 3]')
        if self.host_lengths[index] != P + L:
            self.resize(index, P + L)
        if P:
            self.append(layer, pk, pv, index=index, before=L)
        if L:
            self.append(layer, key, value, index=index, **how)

    def attend(self, layer, query, out=None, n=None, cu_queries=None, causal=False):
        """Attention of `query` [n,H,Q,D] bf16 (H a multiple of the cache's heads; packed [H,T,D] with cu_queries)
        over the keys of the first n windows."""
        n = self.batch if n is None else n
        return paged_attention(query, self.k[layer], self.v[layer], self.table[:n], self.lengths[:n], cu_queries=cu_queries,
                               causal=causal, out=out, k_exponents=self.k_exponents[layer],
                               v_exponents=self.v_exponents[layer], bad=self.bad)
