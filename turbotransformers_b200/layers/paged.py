"""Serving over a pool of cache pages: every sequence of a batch has its own length, its keys and values lie in pages anywhere in a pool, beams share what they
have in common, and new tokens come one, a few, or a chunk of a prompt at a time.

The functions are the operators themselves, on torch tensors; `PagedKVCache` holds the tensors that they work on, for a stack of layers, and `RotaryEmbedding` the
frequencies of rotary positions. One step of a batch whose sequence b has new[b] new tokens, packed one sequence behind the other as rows of q, k, v:

    cache = PagedKVCache(layers=24, pages=20000, sequences=64, max_tokens=4096, kv_heads=8, head_size=128)
    rotary = RotaryEmbedding(128, device="cuda")
    granted = cache.reserve(new)                           # pages for the new tokens: int32 [64] on the device, 0 where there were none
    for layer in ...:
        q = cache.append(layer, k, v, cu_seqlens, q=q, rotary=rotary)
        context = cache.attend(layer, q, cu_seqlens)       # [tokens, heads, head_size]
    cache.advance(new)                                     # of the rows that were granted
    cache.fork(parents)                                    # beams follow their parents; -1 frees a row

A row that was not granted stays as it was: append and attend pass it over (its rows of their outputs are undefined), advance does not count its tokens, and it can
ask again when others have been freed.

Nothing here reads from the device, and with numbers of tokens and parents in int32 tensors nothing waits for it, so that a step can be captured into a graph; those given
as Python lists are copied there first, which waits. What an index outside its table comes to is said in include/ttb.h, and device_status reports it. It is a serving
path: results carry no gradient, as those of the other layers do not. The reference has no counterpart: its decoder concatenates one cache of equally long sequences a step
(multi_headed_attention.cpp:207-231).
"""
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from .._cxx import cxx

__all__ = ['rotary', 'paged_append', 'paged_attention', 'paged_reserve', 'paged_fork', 'paged_copy', 'paged_compact', 'RotaryEmbedding', 'PagedKVCache']

_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_stream = torch._C._cuda_getCurrentRawStream


def _fail(name, why):
    raise ValueError(f"{name} {why}")


def _gpu(t, name):
    device = t.get_device()
    if device < 0:
        raise RuntimeError(f"{name} is not on a CUDA device: this runtime has no CPU path")
    return device


def _rows(t, name, device, dtype, d=None):
    """(rows, heads, head size, elements between rows) of a [tokens, heads, d] tensor whose heads lie side by side."""
    if t.dim() != 3:
        _fail(name, "must be [tokens, heads, head size]")
    (n, heads, width), (row, head, one) = t.shape, t.stride()
    if width and (one != 1 and width > 1 or head != width and heads > 1):
        _fail(name, "must have its heads side by side (strides [any, head size, 1])")
    if d is not None and width != d:
        _fail(name, f"must have heads of {d}")
    if t.dtype != dtype or t.get_device() != device:
        _fail(name, f"must be {dtype} on cuda:{device}")
    return n, heads, width, row if n > 1 else heads * width


def _like(out, x, name, device):
    """Elements between rows of an output, which has its input's shape, dtype and device."""
    if out.shape != x.shape:
        _fail(name, "must be like its input")
    return _rows(out, name, device, x.dtype)[3]


def _index(t, name, n, device, dtype=torch.int32):
    if t.dtype != dtype or t.get_device() != device or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        _fail(name, f"must be a contiguous {dtype} vector of {n} on cuda:{device}")
    return t.data_ptr()


def _freqs(freqs, device):
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous() or freqs.get_device() != device or freqs.shape[0] == 0:
        _fail("freqs", f"must be a contiguous float64 vector on cuda:{device}, of one at least")
    return freqs.data_ptr(), 2 * freqs.shape[0]


def _table(table, device):
    """(address, elements between rows, rows, width) of a page table."""
    if table.dim() != 2 or table.dtype != torch.int32 or table.get_device() != device:
        _fail("table", f"must be int32 [sequences, pages] on cuda:{device}")
    (B, width), (row, one) = table.shape, table.stride()
    if one != 1 and width > 1:
        _fail("table", "must have contiguous rows")
    return table.data_ptr(), row if B > 1 else width, B, width


def _kv(keys, values, table, cu_seqlens, past_lens, room, dtype, device):
    """The arguments that describe one layer's pages."""
    shape, strides = keys.shape, keys.stride()
    if len(shape) != 4 or shape != values.shape:
        _fail("keys and values", "must be [pages, key heads, page tokens, head size], alike")
    if keys.dtype != dtype or values.dtype != dtype or keys.get_device() != device or values.get_device() != device:
        _fail("keys and values", f"must be {dtype} on cuda:{device}, as the rows are")
    pages, heads, tokens, d = shape
    if strides != values.stride() or strides[1:] != (tokens * d, d, 1):
        _fail("keys and values", "must have contiguous pages, equally far apart")
    at, row, B, width = _table(table, device)
    return (keys.data_ptr(), values.data_ptr(), strides[0] if pages > 1 else heads * tokens * d, pages, heads, tokens, d, at, row, width,
            _index(cu_seqlens, "cu_seqlens", B + 1, device), _index(past_lens, "past_lens", B, device), B,
            0 if room is None else _index(room, "room", B, device))


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor, *, interleaved: bool = False, scale: float = 1.0,
           out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None):
    """Rotary positions of q [tokens, heads, d] and k [tokens, key heads, d] (or None): returns (q, k) turned, in new tensors or in `out` (which may be (q, k)
    themselves). positions: int64 [tokens]. freqs: float64 [n], radians a position; the first 2n elements of every head are turned, in pairs (i, i + n), or (2i, 2i + 1) if
    interleaved, and their length is multiplied by scale."""
    device, dtype = _gpu(q, "q"), q.dtype
    if dtype not in _CODE:
        _fail("q", "must be fp32, fp16 or bf16")
    T, heads, d, ldq = _rows(q, "q", device, dtype)
    at, turned = _freqs(freqs, device)
    where = _index(positions, "positions", T, device, torch.int64)
    kp = kv_heads = ldk = 0
    if k is not None:
        n, kv_heads, _, ldk = _rows(k, "k", device, dtype, d)
        if n != T:
            _fail("k", "must have q's tokens")
        kp = k.data_ptr()
    if out is None:
        q_out, k_out = torch.empty_like(q), None if k is None else torch.empty_like(k)
        ldq_out, ldk_out = heads * d, kv_heads * d
    else:
        q_out, k_out = out
        if (k_out is None) != (k is None):
            _fail("out", "must have keys where there are keys")
        ldq_out, ldk_out = _like(q_out, q, "out[0]", device), 0 if k is None else _like(k_out, k, "out[1]", device)
    cxx.rotary(device, _stream(device), _CODE[dtype], q.data_ptr(), kp, q_out.data_ptr(), kp and k_out.data_ptr(), ldq, ldk, ldq_out, ldk_out, T, heads, kv_heads, d,
               turned, where, at, interleaved, scale)
    return q_out, k_out


def paged_append(k: torch.Tensor, v: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, cu_seqlens: torch.Tensor,
                 past_lens: torch.Tensor, *, q: Optional[torch.Tensor] = None, freqs: Optional[torch.Tensor] = None, interleaved: bool = False, scale: float = 1.0,
                 out: Optional[torch.Tensor] = None, room: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Files k and v [tokens, key heads, d] of new tokens as tokens past_lens[b] and following of their sequences. Sequence b's are rows cu_seqlens[b] to
    cu_seqlens[b + 1]; table int32 [sequences, width] lists the pages of each; keys and values are the layer's pool [pages, key heads, page tokens, d]. With `freqs` (see
    rotary) the keys are turned by their places on the way, and so is q, which is returned in a new tensor or in `out`. Sequences with 0 in room (int32 [sequences],
    what paged_reserve granted) are passed over: nothing of them is filed, and their rows of q are not turned."""
    device, dtype = _gpu(k, "k"), k.dtype
    if dtype not in _CODE:
        _fail("k", "must be fp16 or bf16")
    T, heads, d, ldk = _rows(k, "k", device, dtype)
    n, other, _, ldv = _rows(v, "v", device, dtype, d)
    if n != T or other != heads:
        _fail("v", "must be like k")
    kv = _kv(keys, values, table, cu_seqlens, past_lens, room, dtype, device)
    if kv[4] != heads or kv[6] != d:
        _fail("k", "must have the pool's heads")
    if freqs is None:
        if q is not None:
            _fail("q", "is turned by freqs: it has none without them")
        cxx.paged_append(device, _stream(device), _CODE[dtype], *kv, T, k.data_ptr(), ldk, v.data_ptr(), ldv, 0, 0, False, 1.0, 0, 0, 0, 0, 0)
        return None
    at, turned = _freqs(freqs, device)
    qp = op = ldq = ldq_out = q_heads = 0
    if q is not None:
        n, q_heads, _, ldq = _rows(q, "q", device, dtype, d)
        if n != T:
            _fail("q", "must have k's tokens")
        if out is None:
            out, ldq_out = torch.empty_like(q), q_heads * d
        else:
            ldq_out = _like(out, q, "out", device)
        qp, op = q.data_ptr(), out.data_ptr()
    cxx.paged_append(device, _stream(device), _CODE[dtype], *kv, T, k.data_ptr(), ldk, v.data_ptr(), ldv, at, turned, interleaved, scale, qp, op, ldq, ldq_out, q_heads)
    return out if q is not None else None


def paged_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, cu_seqlens: torch.Tensor, past_lens: torch.Tensor, *,
                    causal: bool = True, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    room: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [tokens, heads, d] over the pages of its sequences (arguments as for paged_append, whose new tokens have been filed): token i of a sequence sees its
    cached tokens up to itself, or all past + new of them if not causal. heads is a multiple of the key heads; scale is d ** -0.5 unless given. out does not overlap q. Rows that belong to no sequence,
    or to one with 0 in room (as for paged_append), are left as they are in `out`, undefined without it."""
    device, dtype = _gpu(q, "q"), q.dtype
    if dtype not in _CODE:
        _fail("q", "must be fp16 or bf16")
    T, heads, d, ldq = _rows(q, "q", device, dtype)
    kv = _kv(keys, values, table, cu_seqlens, past_lens, room, dtype, device)
    if kv[6] != d or heads % max(kv[4], 1):
        _fail("q", "must have the pool's head size, and a multiple of its heads")
    if out is None:
        out, ldo = torch.empty_like(q), heads * d
    else:
        ldo = _like(out, q, "out", device)
    cxx.paged_attention(device, _stream(device), _CODE[dtype], *kv, q.data_ptr(), ldq, T, heads, causal, d ** -0.5 if scale is None else scale, out.data_ptr(), ldo)
    return out


def _tables(table, lens, refs):
    device = _gpu(table, "table")
    t = _table(table, device)
    if refs.dim() != 1:
        _fail("refs", "must be a vector")
    pages = refs.shape[0]
    return device, t + (0 if lens is None else _index(lens, "lens", t[2], device), _index(refs, "refs", pages, device), pages)


def _pool(pool):
    shape, strides = pool.shape, pool.stride()
    if len(shape) < 3:
        _fail("pool", "must be [planes, pages, ...]")
    page = 1
    for n, stride in zip(reversed(shape[2:]), reversed(strides[2:])):
        if stride != page and n > 1:
            _fail("pool", "must have contiguous pages")
        page *= n
    size, planes, pages = pool.element_size(), shape[0], shape[1]
    page_stride = strides[1] if pages > 1 else page
    return pool.data_ptr(), planes, size * (strides[0] if planes > 1 else pages * page_stride), pages, size * page_stride, size * page


def paged_reserve(table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, new_tokens: torch.Tensor, page_tokens: int, *, room: Optional[torch.Tensor] = None):
    """Room for new_tokens[b] more tokens of every row of the page table: pages that the row lists already behind its tokens, then the lowest free ones (those of refs 0),
    which are taken into the table. A row that would write to a page that other rows list too gets one of its own in its place. Returns (granted int32 [sequences], copies int32 [sequences, 2]); hand the copies to paged_copy before the new
    tokens are filed. A row that is not granted (0) has been left alone: the pool is full, or its row of the table, or the row or its number of tokens is bad (see device_status).
    room (int32 [sequences]) receives what is granted too: a tensor that is kept from step to step, for paged_append and paged_attention."""
    device, t = _tables(table, lens, refs)
    new = _index(new_tokens, "new_tokens", t[2], device)
    granted, copies = torch.empty_like(new_tokens), new_tokens.new_empty((t[2], 2))
    cxx.paged_reserve(device, _stream(device), *t, new, page_tokens, granted.data_ptr(), copies.data_ptr(), 0 if room is None else _index(room, "room", t[2], device))
    return granted, copies


def paged_fork(table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor) -> None:
    """Row b of the page table becomes what row parents[b] was, and shares its pages; parents[b] = -1 frees the row. table, lens and refs are changed in place."""
    device, t = _tables(table, lens, refs)
    cxx.paged_fork(device, _stream(device), *t, _index(parents, "parents", t[2], device))


def paged_copy(pool: torch.Tensor, pairs: torch.Tensor) -> None:
    """Page pairs[i, 1] of every plane of pool [planes, pages, ...] becomes a copy of page pairs[i, 0] (int32 [n, 2]; pairs with a negative entry are left out). A page that
    is written may not be in another pair."""
    device = _gpu(pool, "pool")
    if pairs.dim() != 2 or pairs.shape[1] != 2 or pairs.dtype != torch.int32 or pairs.get_device() != device or not pairs.is_contiguous():
        _fail("pairs", f"must be a contiguous int32 [n, 2] on cuda:{device}")
    cxx.paged_copy(device, _stream(device), *_pool(pool), pairs.data_ptr(), pairs.shape[0])


def paged_compact(table: torch.Tensor, refs: torch.Tensor, pool: torch.Tensor) -> torch.Tensor:
    """Moves the pages in use to the front of the pool, table and refs with them. Returns how many there are (int32 [1] on the device)."""
    device, t = _tables(table, None, refs)
    if pool.get_device() != device:
        _fail("pool", f"must be on cuda:{device}")
    used = refs.new_empty(1)
    cxx.paged_compact(device, _stream(device), *t, *_pool(pool), used.data_ptr())
    return used


class RotaryEmbedding:
    """Frequencies of rotary positions, base ** (-2i / dim) radians a position for the pairs of the first `dim` elements of a head, and how they are stretched for contexts
    `factor` times as long as the model was trained for:
        None      as they are
        "linear"  all divided by factor (positions are interpolated)
        "ntk"     the base raised, so that the slowest is divided by factor and the fastest stays
        "yarn"    those that turn more than `fast` times in `trained` tokens stay, those that turn less than `slow` times are divided by factor, a ramp over the pairs
                  between; turned elements are scaled by 0.1 ln(factor) + 1
    """

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, stretch: Optional[str] = None, factor: float = 1.0, trained: int = 2048,
                 fast: float = 32.0, slow: float = 1.0, device: Union[str, torch.device] = "cuda"):
        if dim <= 0 or dim % 2:
            raise ValueError("dim must be even and positive")
        if stretch not in (None, "linear", "ntk", "yarn"):
            raise ValueError(f"unknown stretch {stretch!r}")
        if factor < 1.0 and stretch is not None:
            raise ValueError("factor must be at least 1")
        if stretch == "ntk":
            base = base * factor ** (dim / max(dim - 2, 1))
        freqs = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        self.interleaved, self.scale = interleaved, 1.0
        if stretch == "linear":
            freqs = freqs / factor
        elif stretch == "yarn":
            # the pair (as a real number) that turns `turns` times in the trained length
            pair = lambda turns: dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
            ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
            freqs = freqs / factor * ramp + freqs * (1 - ramp)
            self.scale = 0.1 * math.log(factor) + 1.0
        self.freqs = freqs.to(device)

    def __call__(self, q, k, positions, out=None):
        """rotary() of q and k at these positions."""
        return rotary(q, k, positions, self.freqs, interleaved=self.interleaved, scale=self.scale, out=out)


class PagedKVCache:
    """The keys and values of a stack of layers in one pool of pages, and the sequences that they belong to. Row b of the page table is sequence b: `sequences` of them at once,
    a row without tokens being free. `lens` (int32, on the device) are the tokens cached; advance() moves them on when all layers have filed a step's tokens. `room` (int32, on the
    device) is what reserve() granted last, which append(), attend() and advance() go by: 1 for all rows before the first."""

    def __init__(self, layers: int, pages: int, sequences: int, max_tokens: int, kv_heads: int, head_size: int, page_tokens: int = 16,
                 dtype: torch.dtype = torch.float16, device: Union[str, torch.device] = "cuda"):
        if dtype not in (torch.float16, torch.bfloat16):
            raise NotImplementedError("caches are provided for fp16 / bf16 models")
        width = -(-max_tokens // page_tokens)
        self.page_tokens = page_tokens
        self.pool = torch.empty((2 * layers, pages, kv_heads, page_tokens, head_size), dtype=dtype, device=device)
        self.table = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.room = torch.ones(sequences, dtype=torch.int32, device=device)

    def _counts(self, values) -> torch.Tensor:
        return values if isinstance(values, torch.Tensor) else torch.tensor(values, dtype=torch.int32).to(self.table.device)

    def reserve(self, new_tokens: Union[torch.Tensor, Sequence[int]]) -> torch.Tensor:
        """Pages for new_tokens[b] more tokens of every sequence; pages that are shared and about to be written are copied. Returns what paged_reserve grants."""
        granted, copies = paged_reserve(self.table, self.lens, self.refs, self._counts(new_tokens), self.page_tokens, room=self.room)
        paged_copy(self.pool, copies)
        return granted

    def append(self, layer: int, k, v, cu_seqlens, q=None, rotary: Optional[RotaryEmbedding] = None, out=None):
        """paged_append into a layer's pages; with `rotary`, q is returned turned."""
        turn = {} if rotary is None else {"q": q, "freqs": rotary.freqs, "interleaved": rotary.interleaved, "scale": rotary.scale, "out": out}
        if rotary is None and q is not None:
            raise ValueError("q is turned by rotary positions: it has none without them")
        return paged_append(k, v, self.pool[2 * layer], self.pool[2 * layer + 1], self.table, cu_seqlens, self.lens, room=self.room, **turn)

    def attend(self, layer: int, q, cu_seqlens, causal: bool = True, scale: Optional[float] = None, out=None):
        """paged_attention over a layer's pages, between append and advance."""
        return paged_attention(q, self.pool[2 * layer], self.pool[2 * layer + 1], self.table, cu_seqlens, self.lens, causal=causal, scale=scale, out=out,
                               room=self.room)

    def advance(self, new_tokens: Union[torch.Tensor, Sequence[int]]) -> None:
        """The new tokens are cached now, those of the sequences that had room. Fewer than were reserved may be kept: the rest of the room stays the sequence's."""
        self.lens.addcmul_(self.room, self._counts(new_tokens))

    def fork(self, parents: Union[torch.Tensor, Sequence[int]]) -> None:
        """paged_fork: sequence b becomes what parents[b] was; -1 frees it."""
        paged_fork(self.table, self.lens, self.refs, self._counts(parents))

    def release(self, sequences: Union[torch.Tensor, Sequence[int]]) -> None:
        """Frees these sequences' pages (those that no other lists). (A tensor of them is read by the host; fork() takes parents on the device.)"""
        gone = set(sequences.tolist() if isinstance(sequences, torch.Tensor) else sequences)
        self.fork([-1 if b in gone else b for b in range(self.table.shape[0])])

    def compact(self) -> torch.Tensor:
        """paged_compact: the pages in use move to the front of the pool."""
        return paged_compact(self.table, self.refs, self.pool)
