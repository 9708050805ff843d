"""Attention over a paged cache of secret-shared keys and values, for both
parties on one GPU: rotary positions and the append into the cache, the
scores and values of packed sequences (whole prompts and single tokens,
causal, grouped heads), the row max of ragged rows, and the block that runs
them with the softmax block between.

A cached row X is held as the public E = X - B and the dealer's shares B_0,
B_1 of its mask; a call's other operand Y carries a fresh mask A, and the
Beaver product of the two, Z_p = C_p + D B_p + A_p E (+ D E for party 0) with
D = Y - A, needs no new open of the cached side.  A slot that is written again
needs a freshly dealt mask.  The reference keeps its cache as share tensors
(include/nn/kv_cache.hpp) and opens both operands in every product
(src/nn/matmul_beaver.cpp).

All tensors live on the context's device; shares and opened words are int64
tensors (the words of Z_2^64).  Calls are asynchronous on `stream` (default:
the device's current stream); what they are given has to stay allocated until
that stream has passed them, and outputs overlap no input.  Wrong device-side
data (slots, positions, pages) is reported by Context.sync.
"""
from __future__ import annotations

import ctypes as C
import math
import struct

import numpy as np
import torch

from . import _lib
from ._lib import AttnSeqs, RopeAppend, check
from .engine import Context, TruncTables
from .layer import _CoeffGate, _Trunc, load_layer_tables
from .softmax import SoftmaxBlock, load_tables

M64 = (1 << 64) - 1


# -- arguments ----------------------------------------------------------------
# A decode step makes a dozen of these calls on a few thousand words: what the
# checks cost on the host counts there, so they look at one attribute after
# the other and only a refusal formats anything.

_current_raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream(ctx: Context, stream) -> int | None:
    """The raw stream a call runs on (None: the device's legacy stream)."""
    if stream is None:
        return _current_raw(ctx.device) or None
    if isinstance(stream, int):
        return stream or None
    if stream.device_index != ctx.device:
        raise ValueError(f"the stream is on cuda:{stream.device_index}, the context on cuda:{ctx.device}")
    return stream.cuda_stream or None


def _empty(ctx: Context, shape, stream=None, like=None):
    """Words on the context's device, allocated on the stream that writes them
    and kept until the caller's current stream has passed its use of them.
    like: a checked tensor of words there (half the host's time of a new one)."""
    if stream is None:
        if like is not None:
            return like.new_empty(shape)
        return torch.empty(shape, dtype=torch.int64, device=ctx.device)
    now = torch.cuda.current_stream(ctx.device)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=ctx.device) if stream else torch.cuda.default_stream(ctx.device)
    if stream == now:
        return torch.empty(shape, dtype=torch.int64, device=ctx.device)
    with torch.cuda.stream(stream):
        t = torch.empty(shape, dtype=torch.int64, device=ctx.device)
    t.record_stream(now)
    return t


def _elsewhere(ctx: Context, name: str, device: int):
    raise ValueError(f"the {name} is on cuda:{device}, the context on cuda:{ctx.device}")


def _refuse(ctx: Context, name: str, t, shape, dtype):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise ValueError(f"{name}: expected a {dtype} tensor")
    if t.get_device() != ctx.device:
        raise ValueError(f"{name}: on {t.device}, the context is on cuda:{ctx.device}")
    if t.dim() != len(shape) or any(w is not None and w != g for w, g in zip(shape, t.shape)):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple('any' if w is None else w for w in shape)}")
    raise ValueError(f"{name}: not contiguous")


def _want(ctx: Context, name: str, t, shape: tuple, dtype=torch.int64) -> int:
    """The address of a dense tensor: int64 words unless `dtype`, on the device, of the shape (None: any extent)."""
    try:
        if t.dtype is dtype and t.get_device() == ctx.device and t.is_contiguous() and (
                t.shape == shape or (None in shape and t.dim() == len(shape) and
                                     all(w is None or w == g for w, g in zip(shape, t.shape)))):
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(ctx, name, t, shape, dtype)


_Two = C.c_void_p * 2
_TwoWords = C.c_uint64 * 2


def _pair(ctx: Context, name: str, ts, shape: tuple):
    """Both parties' addresses."""
    if not isinstance(ts, (tuple, list)) or len(ts) != 2:
        raise ValueError(f"{name}: expected both parties' tensors")
    x, y = ts
    return _Two(_want(ctx, name, x, shape), _want(ctx, name, y, shape))


def _masks(r):
    try:
        r0, r1 = r
        return _TwoWords(int(r0) & M64, int(r1) & M64)
    except (TypeError, ValueError):
        raise ValueError("r: expected both parties' shares of the mask") from None


# -- rotary tables --------------------------------------------------------------

def rope_table_words(max_pos: int, rot_dim: int, frac_bits: int, base: float = 10000.0, scale: float = 1.0,
                     low_freq: float | None = None, high_freq: float | None = None, trained_pos: int | None = None):
    """Cosines and sines of every position in fixed point: two int32 arrays
    [max_pos][rot_dim / 2], pair i turning by pos * base^(-2i / rot_dim).

    scale > 1 stretches positions for contexts longer than the model was
    trained on: every frequency is divided by it (position interpolation), or,
    with trained_pos and low_freq < high_freq, only those that turn fewer than
    low_freq times over trained_pos positions; frequencies that turn more than
    high_freq times stay, and those between are blended linearly in the number
    of turns.  Angles are formed in 64-bit floats: those of far positions have
    lost nothing that the rounding to frac_bits would keep."""
    if rot_dim < 0 or rot_dim % 2 or max_pos < 1 or not 1 <= frac_bits <= 16 or not base > 0 or not scale > 0:
        raise ValueError("rope_tables: bad size, fractional bits, base or scale")
    half = rot_dim // 2
    inv = base ** (-np.arange(half, dtype=np.float64) / max(half, 1))
    if low_freq is not None or high_freq is not None or trained_pos is not None:
        if low_freq is None or high_freq is None or trained_pos is None or not 0 <= low_freq < high_freq:
            raise ValueError("rope_tables: the blended form takes trained_pos and low_freq < high_freq")
        turns = trained_pos * inv / (2.0 * math.pi)
        keep = np.clip((turns - low_freq) / (high_freq - low_freq), 0.0, 1.0)
        inv = inv * keep + inv / scale * (1.0 - keep)
    else:
        inv = inv / scale
    ang = np.arange(max_pos, dtype=np.float64)[:, None] * inv[None, :]
    one = float(1 << frac_bits)
    return tuple(np.rint(f(ang) * one).astype(np.int32) for f in (np.cos, np.sin))


def rope_tables(ctx: Context, max_pos: int, rot_dim: int, frac_bits: int, **kw):
    """rope_table_words on the context's device, as rope_append_pair takes them."""
    dev = torch.device("cuda", ctx.device)
    return tuple(torch.from_numpy(t).to(dev) for t in rope_table_words(max_pos, rot_dim, frac_bits, **kw))


class TruncPair(_Trunc):
    """A GapARS truncation bundle for both parties with its full-domain tables
    filled (frac_bits 1..16): dealer material that stays resident."""

    def __init__(self, ctx: Context, frac_bits: int, seed: int = 1, stream=None):
        if not 1 <= frac_bits <= 16:
            raise ValueError("TruncPair: 1..16 fractional bits")
        dev = torch.device("cuda", ctx.device)
        super().__init__(ctx, np.random.default_rng(seed), frac_bits, dev)
        self.frac_bits, self.device = frac_bits, ctx.device
        self._full = TruncTables(self.bundles(), dev)
        if self._full.any():
            self._full.fill(ctx, _stream(ctx, stream) or 0)
        torch.cuda.synchronize(dev)  # the tables are read on any stream from here on
        self._args = (_lib.TruncDesc * 2)(*self.desc), _Two(*self.table_ptrs()), _masks(self.r)

    def table_ptrs(self):
        return self._full.ptr(0), self._full.ptr(1)

    def eval_pair(self, ctx: Context, d_xhat, d_y0, d_y1, stream=None):
        """Both parties' truncated shares of the opened x^: lookups in the
        tables (a bundle without queries has none and is evaluated as it is)."""
        if self.device != ctx.device:
            _elsewhere(ctx, "truncation bundle", self.device)
        shape = d_xhat.shape
        for name, t in (("x^", d_xhat), ("y0", d_y0), ("y1", d_y1)):
            _want(ctx, name, t, shape)
        if d_xhat.numel() == 0:
            return
        st = _stream(ctx, stream)
        if not self._full.any():
            return super().eval_pair(ctx, d_xhat, d_y0, d_y1, st or 0)
        check(ctx._L.sufb200_trunc_bundle_eval_pair_tables_dev(
            ctx.h, C.byref(self.desc[0]), C.cast(self.kptr[0], C.c_void_p), C.cast(self.ksz[0], C.c_void_p),
            self._full.ptr(0), C.byref(self.desc[1]), C.cast(self.kptr[1], C.c_void_p),
            C.cast(self.ksz[1], C.c_void_p), self._full.ptr(1), d_xhat.data_ptr(), d_xhat.numel(), d_y0.data_ptr(),
            d_y1.data_ptr(), st))


# -- the cache -------------------------------------------------------------------

class ShareCache:
    """The paged cache of one layer: opened pools ek, ev and the masks' shares
    bk, bv (pairs), each [pages][kv_heads][page_size][head_dim].  Slot = page *
    page_size + place.  The constructor deals fresh masks for every slot; a page
    that is to be written again takes fresh_masks first, or the two openings
    under one mask give away the difference of the rows."""

    def __init__(self, ctx: Context, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, seed: int = 1):
        dev = torch.device("cuda", ctx.device)
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        shape = (pages, kv_heads, page_size, head_dim)

        def words():
            return torch.randint(-(2**63), 2**63 - 1, shape, dtype=torch.int64, device=dev, generator=g)

        self._set(ctx, torch.zeros(shape, dtype=torch.int64, device=dev), (words(), words()),
                  torch.zeros(shape, dtype=torch.int64, device=dev), (words(), words()))
        self._dealer = g

    @classmethod
    def from_tensors(cls, ctx: Context, ek, bk, ev, bv) -> "ShareCache":
        """A cache over pools the caller holds, and whose masks they deal."""
        self = cls.__new__(cls)
        self._set(ctx, ek, bk, ev, bv)
        self._dealer = None
        return self

    def fresh_masks(self, pages, seed: int | None = None):
        """New masks for every slot of the given pages (numbers), on the current
        stream: what was cached there is gone, and so is material dealt for it
        (CachedAttentionPair's triples).  The constructor's dealer goes on from where
        it was; a cache over the caller's pools takes a seed, another one every time."""
        at = np.unique(np.asarray(pages, dtype=np.int64).reshape(-1))
        if at.size and not 0 <= at[0] <= at[-1] < self.pages:
            raise ValueError(f"fresh_masks: pages are numbers from 0 to {self.pages - 1}")
        dev = self.ek.device
        g = self._dealer
        if seed is not None:
            g = torch.Generator(device=dev)
            g.manual_seed(seed)
        if g is None:
            raise ValueError("fresh_masks: a cache over the caller's pools takes a seed")
        at = torch.from_numpy(at).to(dev)
        shape = (at.numel(), self.kv_heads, self.page_size, self.head_dim)
        for pool in (*self.bk, *self.bv):
            pool[at] = torch.randint(-(2**63), 2**63 - 1, shape, dtype=torch.int64, device=dev, generator=g)
        for pool in (self.ek, self.ev):
            pool[at] = 0

    def _set(self, ctx, ek, bk, ev, bv):
        args = self._args = RopeAppend()  # what every append into this cache passes
        args.d_ek = _want(ctx, "ek", ek, (None,) * 4)
        shape = tuple(ek.shape)
        args.d_ev = _want(ctx, "ev", ev, shape)
        args.d_bk, args.d_bv = _pair(ctx, "bk", bk, shape), _pair(ctx, "bv", bv, shape)
        self._pools, self.device = (ek, tuple(bk), ev, tuple(bv)), ctx.device
        self.pages, self.kv_heads, self.page_size, self.head_dim = shape
        if min(shape) < 1 or max(shape) >= 2**31 or self.head_dim % 2 or self.head_dim > 256:
            raise ValueError("cache: empty, past 2^31 pages, or a head size that is not even, 2..256")
        args.pages, args.kv_heads, args.page_size, args.head_dim = shape

    # the pools are fixed: appends keep their addresses
    ek = property(lambda self: self._pools[0])
    bk = property(lambda self: self._pools[1])
    ev = property(lambda self: self._pools[2])
    bv = property(lambda self: self._pools[3])


def _strided(ctx: Context, name: str, ts, shape: tuple):
    """Both parties' addresses and the common strides of [tokens][heads][dim] views (the last axis dense;
    an axis of one entry has any stride)."""
    if not isinstance(ts, (tuple, list)) or len(ts) != 2:
        raise ValueError(f"{name}: expected both parties' tensors")
    x, y = ts
    word, device = torch.int64, ctx.device
    for t in ts:
        try:
            if t.dtype is word and t.get_device() == device and t.shape == shape:
                continue
        except AttributeError:
            pass
        _refuse(ctx, name, t, shape, word)
    ld = x.stride()
    if ld != y.stride():
        ld = tuple(s if n > 1 else 0 for s, n in zip(ld, shape))
        if x.numel() and ld != tuple(s if n > 1 else 0 for s, n in zip(y.stride(), shape)):
            raise ValueError(f"{name}: the parties' strides differ")
    if ld[2] != 1 and x.numel():
        raise ValueError(f"{name}: the head's words must be adjacent")
    return x.data_ptr(), y.data_ptr(), ld[0], ld[1]


# sufb200_rope_append up to d_ek: the shares' addresses and strides, positions,
# slots, cosines, sines, the queries' masks and output
_ROPE_FRONT = struct.Struct("=6Q6q7Q")


def rope_append_pair(ctx: Context, q, k, v, positions, slots, cos, sin, trunc: TruncPair | None, a, cache: ShareCache,
                     d_q=None, *, interleaved: bool = False, stream=None):
    """New tokens' queries, keys and values, both parties' shares [tokens]
    [heads][head_dim] (views of fused rows allowed): queries and keys turned to
    their positions (int32 [tokens]; cos, sin: rope_tables, None with trunc None
    for no rotation) and truncated, keys and values opened against the masks of
    their slots into `cache` (int64 [tokens]; -1: padding, nothing written, all
    others distinct), queries opened against the mask shares a into d_q [tokens]
    [q_heads][head_dim], which is returned.  q, a None: append only."""
    if cache.device != ctx.device:
        _elsewhere(ctx, "cache", cache.device)
    if trunc is not None and trunc.device != ctx.device:
        _elsewhere(ctx, "truncation bundle", trunc.device)
    try:
        tokens, kv, dim = k[0].shape[0], cache.kv_heads, cache.head_dim
        heads = 0 if q is None else q[0].shape[1]
    except (TypeError, IndexError, AttributeError):
        raise ValueError("q, k: expected both parties' tensors [tokens][heads][head_dim]") from None
    if tokens >= 2**31:
        raise ValueError("more than 2^31 tokens in one call")
    if heads + 2 * kv >= 2**31:
        raise ValueError("more than 2^31 heads of a token")
    args = RopeAppend.from_buffer_copy(cache._args)
    k0, k1, k_ts, k_hs = _strided(ctx, "k", k, (tokens, kv, dim))
    v0, v1, v_ts, v_hs = _strided(ctx, "v", v, (tokens, kv, dim))
    q0 = q1 = q_ts = q_hs = a0 = a1 = out = 0
    if q is not None:
        shape = (tokens, heads, dim)
        q0, q1, q_ts, q_hs = _strided(ctx, "q", q, shape)
        a0, a1 = _pair(ctx, "a", a, shape)
        if d_q is None:
            d_q = _empty(ctx, shape, stream, q[0])
        out, args.q_heads = _want(ctx, "d_q", d_q, shape), heads
    at_pos = at_cos = at_sin = 0
    if trunc is not None:
        table = cos.shape if isinstance(cos, torch.Tensor) and cos.dim() == 2 else (None, None)
        at_cos = _want(ctx, "cos", cos, table, torch.int32)
        at_sin = _want(ctx, "sin", sin, table, torch.int32)
        at_pos = _want(ctx, "positions", positions, (tokens,), torch.int32)
        half = table[1]
        if table[0] >= 2**31:
            raise ValueError("tables of more than 2^31 positions")
        if 2 * half > dim:
            raise ValueError(f"the tables turn {2 * half} words of a head of {dim}")
        args.max_pos, args.rot_dim = table[0], 2 * half
        args.trunc, args.d_tables, args.r = trunc._args
    elif cos is not None or sin is not None:
        raise ValueError("rotation needs the truncation bundle")
    _ROPE_FRONT.pack_into(args, 0, q0, q1, k0, k1, v0, v1, q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, at_pos,
                          _want(ctx, "slots", slots, (tokens,)), at_cos, at_sin, a0 or 0, a1 or 0, out)
    args.tokens, args.interleaved = tokens, 1 if interleaved else 0
    check(ctx._L.sufb200_rope_append_pair(ctx.h, C.byref(args), _stream(ctx, stream)))
    return d_q


# -- scores and values -------------------------------------------------------------

class AttnLayout:
    """The packed sequences of an attention call, resident on the device:
    sequence b has q_lens[b] new tokens (its queries, packed one sequence after
    the other) and ctx_lens[b] cached tokens, the new ones included, in the
    pages block_table[b] (int32 [batch][most pages] on the device, or lists).
    Causal rows see what is before them: row (b, head, i) has
    max(0, ctx - q + i + 1) keys; otherwise all ctx.  Rows are packed in
    (sequence, head, query) order: row_lengths() is what SoftmaxBlock and
    RowMaxPlan take, `packed` the words in all, `tokens` the queries."""

    def __init__(self, ctx: Context, q_lens, ctx_lens, block_table, page_size: int, q_heads: int, kv_heads: int,
                 causal: bool = True):
        self.device = ctx.device
        dev = torch.device("cuda", ctx.device)
        q, L = np.asarray(q_lens, dtype=np.int64).reshape(-1), np.asarray(ctx_lens, dtype=np.int64).reshape(-1)
        if q.size != L.size or (q < 0).any() or (L < 0).any():
            raise ValueError("layout: one non-negative query and context length per sequence")
        if kv_heads < 1 or q_heads < kv_heads or q_heads % kv_heads or page_size < 1 or max(q_heads, page_size) >= 2**31:
            raise ValueError("layout: query heads must be a multiple of key heads, the page size positive")
        if not isinstance(block_table, torch.Tensor):
            rows = [list(r) for r in block_table]
            wide = np.zeros((len(rows), max([len(r) for r in rows] + [1])), dtype=np.int32)
            for i, r in enumerate(rows):
                if i < q.size and len(r) * page_size < L[i]:
                    raise ValueError("layout: a sequence is longer than its pages")
                if any(not 0 <= pg < 2**31 for pg in r):
                    raise ValueError("layout: pages are numbers from 0 on")
                wide[i, :len(r)] = r
            block_table = torch.from_numpy(wide).to(dev)
        if block_table.dim() != 2:
            raise ValueError("layout: the block table is [batch][most pages]")
        _want(ctx, "block_table", block_table, (q.size, None), torch.int32)
        self.q_lens, self.ctx_lens, self.causal = q, L, bool(causal)
        self.q_heads, self.kv_heads, self.page_size = int(q_heads), int(kv_heads), int(page_size)
        self.tokens, self.batch = int(q.sum()), int(q.size)
        if causal:  # the lengths of a head's rows are consecutive: their sum is a difference of triangles
            first = np.maximum(L - q, 0)
            words = (L * (L + 1) - first * (first + 1)) // 2
        else:
            words = q * L
        base = np.concatenate([[0], np.cumsum(words * q_heads)])
        self.packed = int(base[-1])
        if self.batch and int(L.max()) > block_table.shape[1] * page_size:
            raise ValueError("layout: a sequence is longer than its pages")
        if max(self.tokens, self.batch, int(L.sum()), block_table.shape[1]) >= 2**31:
            raise ValueError("layout: more than 2^31 tokens, or pages of a sequence")
        self._cu = torch.from_numpy(np.concatenate([[0], np.cumsum(q)]).astype(np.int32)).to(dev)
        self._ctx = torch.from_numpy(np.concatenate([[0], np.cumsum(L)]).astype(np.int32)).to(dev)
        self._base = torch.from_numpy(base[:-1].astype(np.int64)).to(dev)
        self._table = block_table
        s = self._seqs = AttnSeqs()
        s.d_cu_q, s.d_cu_ctx, s.d_row_base = self._cu.data_ptr(), self._ctx.data_ptr(), self._base.data_ptr()
        s.d_block_table = block_table.data_ptr()
        s.tokens, s.cached, s.packed = self.tokens, int(L.sum()), self.packed
        s.batch, s.max_pages = self.batch, int(block_table.shape[1])
        s.page_size, s.q_heads, s.kv_heads, s.causal = self.page_size, self.q_heads, self.kv_heads, int(self.causal)
        s.min_q, s.max_q, s.max_ctx = int(q[q > 0].min(initial=2**31 - 1)), int(q.max(initial=0)), int(L.max(initial=0))
        s.min_q = min(s.min_q, s.max_q)
        longest, most = self._bounds()
        if longest and most:  # of one kind alone, max_ctx and max_q say the same
            s.long_ctx, s.short_rows = longest, most
        tiles = self._tile_list()
        if len(tiles):
            self._tiles = torch.from_numpy(tiles).to(dev)
            s.d_tiles, s.n_tiles = self._tiles.data_ptr(), len(tiles)
            places = self._plane_keys()
            if places is not None:
                self._places = torch.from_numpy(places).to(dev)
                s.d_plane_keys, s.plane_keys = self._places.data_ptr(), max(int(places[-1]), _lib.ATTN_KEY_TILE)

    def _tile_list(self) -> np.ndarray:
        """(sequence, row tile) of the sequences with many rows, the longest rows first."""
        group = self.q_heads // self.kv_heads
        rows = self.q_lens * group
        long_ = np.flatnonzero(rows > _lib.ATTN_FEW_ROWS)
        if not len(long_):
            return np.zeros((0, 2), dtype=np.int32)
        count = -(-rows[long_] // _lib.ATTN_ROW_TILE)
        seq = np.repeat(long_, count)
        tile = np.arange(len(seq)) - np.repeat(np.cumsum(count) - count, count)
        last = (np.minimum((tile + 1) * _lib.ATTN_ROW_TILE, rows[seq]) - 1) // group  # the tile's last query
        length = self.ctx_lens[seq] + (last + 1 - self.q_lens[seq] if self.causal else 0)
        order = np.argsort(-length, kind="stable")
        return np.stack([seq, tile], axis=1)[order].astype(np.int32)

    def _bounds(self) -> tuple[int, int]:
        """The longest context of the sequences with many rows, the most rows of the others."""
        rows = self.q_lens * (self.q_heads // self.kv_heads)
        many = rows > _lib.ATTN_FEW_ROWS
        return int(self.ctx_lens[many].max(initial=0)), int(rows[~many].max(initial=0))

    def _plane_keys(self) -> np.ndarray | None:
        """Where the cached tokens of the sequences with many rows lie in the products' workspace (prefix
        sums, whole key tiles); None where those are all sequences there are, or past 32 bits."""
        long_ = self.q_lens * (self.q_heads // self.kv_heads) > _lib.ATTN_FEW_ROWS
        if not self.ctx_lens[~long_].any():
            return None
        tile = _lib.ATTN_KEY_TILE
        at = np.concatenate([[0], np.cumsum(np.where(long_, -(-self.ctx_lens // tile) * tile, 0))])
        return at.astype(np.int32) if at[-1] < 2**31 - tile else None

    def row_lengths(self) -> np.ndarray:
        """Keys of every row, in (sequence, head, query) order."""
        out = [np.tile(np.maximum(0, L - n + 1 + np.arange(n)) if self.causal else np.full(n, L), self.q_heads)
               for n, L in zip(self.q_lens, self.ctx_lens)]
        return np.concatenate(out).astype(np.int64) if out else np.zeros(0, dtype=np.int64)

    def _for_pool(self, ctx, name, e, b):
        """(the sequences with the pool's sizes, the pool's address, its masks' addresses)"""
        if self.device != ctx.device:
            _elsewhere(ctx, "layout", self.device)
        e_ptr = _want(ctx, name, e, (None, self.kv_heads, self.page_size, None))
        shape = e.shape
        pages, _, _, dim = shape
        if pages >= 2**31 or dim >= 2**31:
            raise ValueError(f"{name}: past 2^31 pages")
        s = AttnSeqs.from_buffer_copy(self._seqs)
        s.pages, s.head_dim = pages, dim
        return s, e_ptr, _pair(ctx, f"{name}'s masks", b, shape)


def attn_scores_pair(ctx: Context, d_q, a, c, r, ek, bk, layout: AttnLayout, out=None, stream=None):
    """The opened, masked scores of every packed (row, key): the opened queries
    d_q and their mask's shares a [tokens][q_heads][head_dim], the packed shares
    c of the triple's product, r the shares of the output's mask, ek and bk a
    cache's keys.  Returns x^ [packed]."""
    seqs, e, b = layout._for_pool(ctx, "ek", ek, bk)
    shape, packed = (layout.tokens, layout.q_heads, seqs.head_dim), (layout.packed,)
    if out is None:
        out = _empty(ctx, layout.packed, stream, ek)
    check(ctx._L.sufb200_attn_scores_pair(ctx.h, C.byref(seqs), _want(ctx, "d_q", d_q, shape),
                                          _pair(ctx, "a", a, shape), _pair(ctx, "c", c, packed), _masks(r), e, b,
                                          _want(ctx, "out", out, packed), _stream(ctx, stream)))
    return out


def attn_values_pair(ctx: Context, p, a, c, r, ev, bv, layout: AttnLayout, out=None, stream=None):
    """The opened, masked value products of every query and head: the packed
    shares p of the probabilities and a of their mask, the shares c of the
    triple's product [tokens][q_heads][head_dim], ev and bv a cache's values.
    Returns x^ [tokens][q_heads][head_dim]."""
    seqs, e, b = layout._for_pool(ctx, "ev", ev, bv)
    shape, packed = (layout.tokens, layout.q_heads, seqs.head_dim), (layout.packed,)
    if out is None:
        out = _empty(ctx, shape, stream, ev)
    check(ctx._L.sufb200_attn_values_pair(ctx.h, C.byref(seqs), _pair(ctx, "p", p, packed),
                                          _pair(ctx, "a", a, packed), _pair(ctx, "c", c, shape), _masks(r), e, b,
                                          _want(ctx, "out", out, shape), _stream(ctx, stream)))
    return out


# -- the row max of ragged rows -----------------------------------------------------

class RowMaxPlan:
    """The rounds of the row-max tournament over packed rows of the given
    lengths: off[k] the device row offsets of round k, pairs[k] its pairs,
    values[k] its packed values, `rounds` how often the longest row halves."""

    def __init__(self, ctx: Context, row_lengths):
        self.device = ctx.device
        dev = torch.device("cuda", ctx.device)
        w = np.asarray(row_lengths, dtype=np.int64).reshape(-1)
        if (w < 0).any() or int(w.max(initial=0)) > 2**30 or int(w.sum()) >= 2**31:
            raise ValueError("rowmax: row lengths must be 0..2^30, below 2^31 words in all")
        self.rows = int(w.size)
        self.off, self.values, self.pairs, self.widths = [], [], [], []
        while True:
            self.off.append(torch.from_numpy(np.concatenate([[0], np.cumsum(w)]).astype(np.int32)).to(dev))
            self.values.append(int(w.sum()))
            self.widths.append(int(w.max(initial=0)))
            if self.widths[-1] <= 1:
                break
            self.pairs.append(int((w // 2).sum()))
            w = (w + 1) // 2
        self.rounds = len(self.pairs)
        self._off = [t.data_ptr() for t in self.off]


def rowmax_open_pair(ctx: Context, plan: RowMaxPlan, c, r, out=None, stream=None):
    """x^ [pairs[0]]: the opened differences of the first round's pairs of c (packed shares)."""
    if plan.device != ctx.device:
        _elsewhere(ctx, "row max plan", plan.device)
    n = plan.pairs[0] if plan.rounds else 0
    words = _pair(ctx, "c", c, (plan.values[0],))
    if out is None:
        out = _empty(ctx, n, stream, c[0])
    o = _want(ctx, "out", out, (n,))
    if n:
        check(ctx._L.sufb200_rowmax_open_pair(ctx.h, words, plan.rows, plan.widths[0], plan._off[0], plan._off[1],
                                              _masks(r), o, _stream(ctx, stream)))
    return out


def rowmax_round_pair(ctx: Context, plan: RowMaxPlan, k: int, c, relu, r_next=None, nxt=None, out=None, stream=None):
    """Round k: its values c (packed shares) and the gate's shares relu of its
    pairs to the next round's values, and, with r_next, the open of their
    differences.  Returns ((next_0, next_1), x^ or None)."""
    if plan.device != ctx.device:
        _elsewhere(ctx, "row max plan", plan.device)
    if not 0 <= k < plan.rounds:
        raise ValueError(f"rowmax: round {k} of {plan.rounds}")
    n, more = plan.values[k + 1], k + 1 < plan.rounds
    words, gates = _pair(ctx, "c", c, (plan.values[k],)), _pair(ctx, "relu", relu, (plan.pairs[k],))
    if nxt is None:
        nxt = _empty(ctx, n, stream, c[0]), _empty(ctx, n, stream, c[0])
        to = _Two(nxt[0].data_ptr(), nxt[1].data_ptr())
    else:
        to = _pair(ctx, "next", nxt, (n,))
    o = off2 = r = None
    if r_next is not None:
        if not more:
            raise ValueError("rowmax: the last round has no further differences to open")
        if out is None:
            out = _empty(ctx, plan.pairs[k + 1], stream, c[0])
            o = out.data_ptr()
        else:
            o = _want(ctx, "out", out, (plan.pairs[k + 1],))
        off2, r = plan._off[k + 2], _masks(r_next)
    check(ctx._L.sufb200_rowmax_round_pair(
        ctx.h, words, gates, plan.rows, plan.widths[k], plan._off[k], plan._off[k + 1], off2, r, to, o,
        _stream(ctx, stream)))
    return nxt, out if r_next is not None else None


def maxdiff_ragged_pair(ctx: Context, plan: RowMaxPlan, m, s, out=None, stream=None):
    """t_p = max_p[row] - s_p over the packed rows: m the last round's values, s the first's."""
    if plan.device != ctx.device:
        _elsewhere(ctx, "row max plan", plan.device)
    n = (plan.values[0],)
    top, words = _pair(ctx, "max", m, (plan.values[-1],)), _pair(ctx, "s", s, n)
    if out is None:
        out = _empty(ctx, n, stream, s[0]), _empty(ctx, n, stream, s[0])
    check(ctx._L.sufb200_maxdiff_ragged_pair(ctx.h, top, words, plan.rows, plan.widths[0], plan._off[0], plan._off[-1],
                                             _pair(ctx, "out", out, n), _stream(ctx, stream)))
    return out


# -- the block ------------------------------------------------------------------------

class CachedAttentionPair:
    """One attention step over a cache for both parties: the new tokens
    appended with their rotary positions, causal scores against everything
    cached, the row max, the softmax block and the value products, every
    truncation a GapARS bundle.  The constructor deals the step's material for
    the layout (masks, triples, gates; f from the softmax tables); in a
    deployment each step takes freshly dealt material.

    score_shift: bits of 1/sqrt(head_dim) folded into the scores' truncation;
    default log2(sqrt(head_dim)) for head sizes 4^k, otherwise fold the scale
    into the query weights and pass 0."""

    def __init__(self, ctx: Context, cache: ShareCache, layout: AttnLayout, seed: int = 1,
                 score_shift: int | None = None, rope: tuple | None = None, interleaved: bool = False):
        for name, what in (("cache", cache), ("layout", layout)):
            if what.device != ctx.device:
                _elsewhere(ctx, name, what.device)
        if layout.kv_heads != cache.kv_heads or layout.page_size != cache.page_size:
            raise ValueError("attention: the layout's heads or pages are not the cache's")
        dim = cache.head_dim
        if score_shift is None:
            score_shift = (dim.bit_length() - 1) // 2
            if 4**score_shift != dim:
                raise ValueError("attention: 1/sqrt(head_dim) is not a power of two: pass score_shift")
        self.ctx, self.cache, self.layout, self.rope, self.interleaved = ctx, cache, layout, rope, interleaved
        sm_tables = load_tables()
        f = self.frac_bits = int(sm_tables["frac_bits"])
        rng = np.random.default_rng(seed)

        def sub():
            return int(rng.integers(1, 2**62))

        dev = torch.device("cuda", ctx.device)
        g = torch.Generator(device=dev)
        g.manual_seed(sub())

        def words(*shape):
            return torch.randint(-(2**63), 2**63 - 1, shape, dtype=torch.int64, device=dev, generator=g)

        T, H = layout.tokens, layout.q_heads
        self.tr_rope = TruncPair(ctx, f, sub()) if rope is not None else None
        self.tr_s, self.tr_o = TruncPair(ctx, f + score_shift, sub()), TruncPair(ctx, f, sub())
        self.a_q = (words(T, H, dim), words(T, H, dim))
        self.a_p = (words(layout.packed), words(layout.packed))
        # the triples' products A B: a product with D = A and E = 0
        zero_e = torch.zeros_like(cache.ek)
        z_q, z_p = torch.zeros_like(self.a_q[0]), torch.zeros_like(self.a_p[0])
        cs = attn_scores_pair(ctx, self.a_q[0] + self.a_q[1], (z_q, z_q), (z_p, z_p), (0, 0), zero_e, cache.bk, layout)
        cv = attn_values_pair(ctx, (self.a_p[0] + self.a_p[1], z_p), (z_p, z_p), (z_q, z_q), (0, 0), zero_e, cache.bv,
                              layout)
        s0, v0 = words(layout.packed), words(T, H, dim)
        self.c_s, self.c_v = (s0, cs - s0), (v0, cv - v0)
        if layout.packed:
            lens = layout.row_lengths()
            self.plan = RowMaxPlan(ctx, lens)
            relu = load_layer_tables()["relu"]
            self.gates = [_CoeffGate(rng, relu) for _ in range(self.plan.rounds)]
            self.softmax = SoftmaxBlock(ctx, lens, seed=sub(), tables=sm_tables)
        ctx.sync(_stream(ctx, None) or 0)

    def run(self, q, k, v, positions, slots, stream=None, trace: dict | None = None):
        """Both parties' shares of the new tokens' queries, keys and values
        [tokens][heads][head_dim] (views of fused rows allowed), their positions
        (None without rotary tables) and cache slots -> both parties' shares of
        the attention output [tokens][q_heads][head_dim]."""
        ctx, layout, st = self.ctx, self.layout, stream

        def new(n):
            return _empty(ctx, n, st), _empty(ctx, n, st)

        raw = _stream(ctx, stream) or 0  # the softmax block and the gates take torch's current device otherwise
        cos, sin = self.rope if self.rope is not None else (None, None)
        d_q = rope_append_pair(ctx, q, k, v, positions, slots, cos, sin, self.tr_rope, self.a_q, self.cache,
                               interleaved=self.interleaved, stream=st)
        p = new(layout.packed)
        if layout.packed:
            xs = attn_scores_pair(ctx, d_q, self.a_q, self.c_s, self.tr_s.r, self.cache.ek, self.cache.bk, layout,
                                  stream=st)
            s = new(layout.packed)
            self.tr_s.eval_pair(ctx, xs, *s, stream=st)
            cur, plan = s, self.plan
            xh = rowmax_open_pair(ctx, plan, cur, self.gates[0].r, stream=st) if plan.rounds else None
            for i, gate in enumerate(self.gates):
                relu = new(plan.pairs[i])
                gate.eval_pair(ctx, xh, *relu, raw)
                nxt = self.gates[i + 1].r if i + 1 < plan.rounds else None
                cur, xh = rowmax_round_pair(ctx, plan, i, cur, relu, nxt, stream=st)
            t = maxdiff_ragged_pair(ctx, plan, cur, s, stream=st)
            self.softmax.run(*t, *p, stream=raw)
            if trace is not None:
                trace.update(d_q=d_q, scores=s, t=t, probs=p)
        xo = attn_values_pair(ctx, p, self.a_p, self.c_v, self.tr_o.r, self.cache.ev, self.cache.bv, layout, stream=st)
        o = new(tuple(xo.shape))
        if xo.numel():
            self.tr_o.eval_pair(ctx, xo, *o, stream=st)
        return o
