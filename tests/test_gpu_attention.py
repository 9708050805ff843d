"""Attention over a paged cache of shares against its definition in 64-bit
words, bit for bit (every result is a whole word mod 2^64: tolerance zero):
the rotary append, the scores, the values, the ragged row max, and the block
that runs them together against the plaintext model."""
from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import from_dev, rand_u64, to_dev

pytestmark = pytest.mark.gpu

U = np.uint64
GUARD = 7  # words behind an output that must stay as they were


def _words(rng, *shape):
    return rand_u64(rng, int(np.prod(shape))).reshape(shape)


def _dev(torch, a):
    return to_dev(torch, a)


# -- rotary append ----------------------------------------------------------------

def _turn(x, cos, sin, rot, f, interleaved):
    """x [heads][dim] signed -> rotated and floored, in numpy's int64."""
    half = rot // 2
    y = x.copy()
    i1 = np.arange(half) * 2 if interleaved else np.arange(half)
    i2 = i1 + 1 if interleaved else i1 + half
    y[:, i1] = (x[:, i1] * cos - x[:, i2] * sin) >> f
    y[:, i2] = (x[:, i2] * cos + x[:, i1] * sin) >> f
    return y


ROPE = [  # tokens, q heads, kv heads, dim, rot, interleaved, page, f, bits of the values, padding
    (1, 1, 1, 2, 2, False, 1, 12, 20, 0),
    (1, 12, 12, 64, 64, False, 64, 12, 40, 0),
    (5, 8, 2, 64, 64, True, 16, 12, 40, 2),
    (33, 6, 3, 40, 22, False, 7, 12, 30, 1),
    (33, 6, 3, 40, 22, True, 7, 16, 40, 0),
    (130, 4, 1, 256, 128, False, 100, 8, 45, 3),
    (7, 0, 2, 32, 32, False, 5, 12, 20, 0),  # append only
    (9, 4, 4, 72, 0, False, 4, 12, 60, 1),   # nothing turned
    (64, 4, 2, 128, 128, True, 32, 1, 50, 0),
    (300, 32, 8, 128, 128, False, 64, 12, 44, 0),
    (40, 3, 1, 18, 6, True, 3, 15, 40, 0),
]


def _rope_case(ctx, torch, case, seed, strided=True):
    from suf_b200.attention import ShareCache, TruncPair, rope_tables

    T, hq, hkv, dh, rot, inter, page, f, bits, pad = case
    rng = np.random.default_rng(seed)
    width = (hq + 2 * hkv) * dh
    x = rng.integers(-(2**bits) + 1, 2**bits, (T, width), dtype=np.int64)
    x[0, :4] = [2**bits - 1, -(2**bits) + 1, 0, -1][:x.shape[1]] if width >= 4 else x[0, :4]
    s0 = _words(rng, T, width)
    shares = (s0, x.view(U) - s0)
    ld = width + 3 if strided else width  # rows of a wider buffer: odd strides
    fused = []
    for s in shares:
        buf = np.zeros((T, ld), dtype=U)
        buf[:, :width] = s
        fused.append(_dev(torch, buf)[:, :width].unflatten(1, (hq + 2 * hkv, dh)))
    q = tuple(b[:, :hq] for b in fused) if hq else None
    k, v = tuple(b[:, hq:hq + hkv] for b in fused), tuple(b[:, hq + hkv:] for b in fused)
    pages = -(-T // page) + 2
    pools = [_words(rng, pages, hkv, page, dh) for _ in range(6)]
    d_pools = [_dev(torch, p) for p in pools]
    cache = ShareCache.from_tensors(ctx, d_pools[0], (d_pools[1], d_pools[2]), d_pools[3], (d_pools[4], d_pools[5]))
    slots = rng.permutation(pages * page)[:T].astype(np.int64)
    if pad:
        slots[T - pad:] = -1
    pos = rng.integers(0, 500, T).astype(np.int32)
    pos[0] = 499
    trunc = TruncPair(ctx, f, seed=seed) if rot else None
    cos, sin = rope_tables(ctx, 500, rot, f) if rot else (None, None)
    a = (_words(rng, T, hq, dh), _words(rng, T, hq, dh)) if hq else None
    d_q = torch.full((T, hq, dh), 77, dtype=torch.int64, device="cuda") if hq else None
    hc, hs = (t.cpu().numpy().astype(np.int64) for t in (cos, sin)) if rot else (None, None)
    want_q, want = np.full((T, hq, dh), 77, dtype=np.int64).view(U), [pools[0].copy(), pools[3].copy()]
    for t in range(T):
        if slots[t] < 0:
            continue
        h = x[t].reshape(-1, dh)
        y = h.copy()
        if rot:
            y[:hq + hkv] = _turn(h[:hq + hkv], hc[pos[t]], hs[pos[t]], rot, f, inter)
        pg, at = divmod(int(slots[t]), page)
        if hq:
            want_q[t] = y[:hq].view(U) - a[0][t] - a[1][t]
        want[0][pg, :, at] = y[hq:hq + hkv].view(U) - pools[1][pg, :, at] - pools[2][pg, :, at]
        want[1][pg, :, at] = y[hq + hkv:].view(U) - pools[4][pg, :, at] - pools[5][pg, :, at]
    da = tuple(_dev(torch, m) for m in a) if hq else None
    args = (q, k, v, torch.from_numpy(pos).cuda() if rot else None, torch.from_numpy(slots).cuda(), cos, sin, trunc,
            da, cache, d_q)
    return args, dict(interleaved=inter), (want_q, want[0], want[1]), (d_q, d_pools[0], d_pools[3]), trunc


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("case", ROPE)
def test_rope_append_matches_definition(ctx, torch_cuda, case, strided):
    from suf_b200.attention import rope_append_pair

    args, kw, want, got, _ = _rope_case(ctx, torch_cuda, case, seed=3 + strided, strided=strided)
    rope_append_pair(ctx, *args, **kw)
    ctx.sync()
    for w, g in zip(want, got):
        if g is not None:
            assert (from_dev(g) == w).all()


def test_rope_append_with_a_carry_free_bundle(ctx, torch_cuda):
    """A mask whose low bits are zero has no carry queries and no tables."""
    from suf_b200.attention import TruncPair, rope_append_pair

    seed = next(s for s in range(200) if int(TruncPair(ctx, 1, seed=s).desc[0].nq) == 0)
    args, kw, want, got, trunc = _rope_case(ctx, torch_cuda, (6, 4, 2, 32, 32, False, 8, 1, 40, 0), seed)
    assert trunc.table_ptrs() == (None, None)
    rope_append_pair(ctx, *args, **kw)
    ctx.sync()
    assert all((from_dev(g) == w).all() for w, g in zip(want, got))


def test_rope_append_reports_bad_slots_and_positions(ctx, torch_cuda):
    from suf_b200 import SufB200Error
    from suf_b200.attention import rope_append_pair

    for what in ("slot", "position"):
        args, kw, want, got, _ = _rope_case(ctx, torch_cuda, (6, 4, 2, 32, 32, False, 8, 12, 40, 0), 5)
        args = list(args)
        for bad in ((8 * 3, -2, 2**40) if what == "slot" else (500, -1, 2**31 - 1)):
            i = 4 if what == "slot" else 3
            args[i] = args[i].clone()
            args[i][2] = bad
            rope_append_pair(ctx, *args, **kw)
            with pytest.raises(SufB200Error):
                ctx.sync()
            ctx.sync()  # reported once
        keep = [0, 1, 3, 4, 5]
        assert (from_dev(got[0])[keep] == want[0][keep]).all()  # the other tokens are done


# -- scores and values ---------------------------------------------------------------

ATTN = [  # (new tokens, context) per sequence, q heads, kv heads, dim, page, causal
    ([(1, 1)], 1, 1, 2, 1, True),
    ([(1, 129)], 12, 12, 64, 64, True),
    ([(1, 300), (1, 1), (1, 77)], 8, 2, 128, 16, True),
    ([(1, 65), (0, 40), (1, 0), (1, 64)], 16, 2, 40, 7, True),   # a sequence without queries, one without keys
    ([(1, 700)], 10, 2, 256, 100, True),                          # groups of five
    ([(3, 50), (2, 2)], 8, 4, 64, 16, True),                      # a few rows
    ([(5, 3), (4, 9)], 6, 3, 72, 5, True),                        # queries that see nothing
    ([(17, 40), (1, 33), (20, 20)], 4, 1, 64, 32, True),          # tiles
    ([(70, 65)], 2, 2, 18, 8, True),
    ([(130, 200), (1, 5)], 4, 2, 96, 64, True),
    ([(128, 128)], 3, 3, 64, 64, False),
    ([(3, 40), (1, 9)], 4, 2, 64, 16, False),
    ([(200, 333), (64, 64), (129, 129)], 8, 2, 128, 48, True),
    ([(33, 260)], 2, 1, 256, 64, False),
    ([(1, 5000), (1, 4097)], 4, 4, 80, 64, True),                 # long rows, split
    ([(40, 2100)], 4, 2, 32, 64, True),
    ([(20, 4500), (1, 4097)], 2, 1, 64, 64, True),                # tiles over more keys than one exact accumulation
    ([(9, 130), (10, 9)], 3, 3, 34, 16, True),                    # just past the row kernels, empty rows
    ([(1, 256), (1, 255)], 4, 1, 128, 64, True),                  # one CTA's whole context
    ([(1, 257)], 8, 1, 62, 64, True),
    ([(40, 60), (1, 300), (2, 1)], 4, 2, 160, 16, True),          # prompts and single tokens, wide heads
    ([(1, 300), (40, 60), (0, 5), (3, 0), (20, 7)], 6, 2, 64, 32, False),
]


class _Attn:
    def __init__(self, ctx, torch, case, seed):
        from suf_b200.attention import AttnLayout

        seqs, hq, hkv, dh, page, causal = case
        rng = np.random.default_rng(seed)
        self.q, self.L = [n for n, _ in seqs], [c for _, c in seqs]
        self.T, self.hq, self.hkv, self.dh, self.page = sum(self.q), hq, hkv, dh, page
        need = [-(-c // page) for c in self.L]
        self.pages = sum(need) + 2
        order = rng.permutation(self.pages)
        self.table, at = [], 0
        for n in need:
            self.table.append([int(p) for p in order[at:at + n]])
            at += n
        self.e, self.b0, self.b1 = (_words(rng, self.pages, hkv, page, dh) for _ in range(3))
        self.r = tuple(int(v) for v in rand_u64(rng, 2))
        self.layout = AttnLayout(ctx, self.q, self.L, self.table, page, hq, hkv, causal=causal)
        self.lens = [[max(0, c - n + i + 1) if causal else c for i in range(n)] for n, c in seqs]
        self.n = sum(sum(x) for x in self.lens) * hq
        self.torch, self.rng = torch, rng
        self.pool = (_dev(torch, self.e), (_dev(torch, self.b0), _dev(torch, self.b1)))

    def seq(self, b, h):
        j = np.arange(self.L[b])
        ids = np.array(self.table[b], dtype=np.int64)[j // self.page] if self.L[b] else j
        return [x[ids, h // (self.hq // self.hkv), j % self.page] for x in (self.e, self.b0, self.b1)]

    def scores(self):
        """(device arguments, expected words)"""
        rng = self.rng
        d, a0, a1 = (_words(rng, self.T, self.hq, self.dh) for _ in range(3))
        c0, c1 = _words(rng, self.n), _words(rng, self.n)
        out, at, t0 = np.zeros(self.n, dtype=U), 0, 0
        for b, n in enumerate(self.q):
            for h in range(self.hq):
                e, b0, b1 = self.seq(b, h)
                for i in range(n):
                    m = self.lens[b][i]
                    dd, w = d[t0 + i, h], slice(at, at + m)
                    z0 = c0[w] + b0[:m] @ dd + e[:m] @ a0[t0 + i, h] + e[:m] @ dd
                    z1 = c1[w] + b1[:m] @ dd + e[:m] @ a1[t0 + i, h]
                    out[w] = (z0 + U(self.r[0])) + (z1 + U(self.r[1]))
                    at += m
            t0 += n
        t = self.torch
        return (_dev(t, d), (_dev(t, a0), _dev(t, a1)), (_dev(t, c0), _dev(t, c1)), self.r, *self.pool,
                self.layout), out

    def values(self):
        rng = self.rng
        p0, p1, a0, a1 = (_words(rng, self.n) for _ in range(4))
        c0, c1 = (_words(rng, self.T, self.hq, self.dh) for _ in range(2))
        out, at, t0 = np.zeros((self.T, self.hq, self.dh), dtype=U), 0, 0
        for b, n in enumerate(self.q):
            for h in range(self.hq):
                e, b0, b1 = self.seq(b, h)
                for i in range(n):
                    m = self.lens[b][i]
                    w = slice(at, at + m)
                    dd = (p0[w] - a0[w]) + (p1[w] - a1[w])
                    z0 = c0[t0 + i, h] + dd @ b0[:m] + a0[w] @ e[:m] + dd @ e[:m]
                    z1 = c1[t0 + i, h] + dd @ b1[:m] + a1[w] @ e[:m]
                    out[t0 + i, h] = (z0 + U(self.r[0])) + (z1 + U(self.r[1]))
                    at += m
            t0 += n
        t = self.torch
        return ((_dev(t, p0), _dev(t, p1)), (_dev(t, a0), _dev(t, a1)), (_dev(t, c0), _dev(t, c1)), self.r,
                *self.pool, self.layout), out


def _guarded(torch, want):
    """An output buffer with guard words behind it, as a dense view of its front."""
    buf = torch.full((want.size + GUARD,), 77, dtype=torch.int64, device="cuda")
    return buf, buf[:want.size].view(want.shape)


@pytest.mark.parametrize("case", ATTN)
def test_scores_match_definition(ctx, torch_cuda, case):
    from suf_b200.attention import attn_scores_pair

    args, want = _Attn(ctx, torch_cuda, case, 11).scores()
    buf, out = _guarded(torch_cuda, want)
    attn_scores_pair(ctx, *args, out=out)
    ctx.sync()
    assert (from_dev(out) == want).all() and (buf[want.size:] == 77).all()


@pytest.mark.parametrize("case", ATTN)
def test_values_match_definition(ctx, torch_cuda, case):
    from suf_b200.attention import attn_values_pair

    args, want = _Attn(ctx, torch_cuda, case, 12).values()
    buf, out = _guarded(torch_cuda, want)
    for _ in range(2):  # a second call on the same buffers gives the same words
        attn_values_pair(ctx, *args, out=out)
        ctx.sync()
        assert (from_dev(out) == want).all() and (buf[want.size:] == 77).all()


@pytest.mark.parametrize("which", ["scores", "values"])
@pytest.mark.parametrize("case", [ATTN[7], ATTN[12], ATTN[20], ATTN[21]])
def test_attention_without_a_tile_list(ctx, torch_cuda, which, case):
    """The C entry's form without an order of work: the same words."""
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, case, 14)
    args, want = getattr(A, which)()
    assert A.layout._seqs.n_tiles > 0
    A.layout._seqs.d_tiles, A.layout._seqs.n_tiles = None, 0
    got = getattr(at, f"attn_{which}_pair")(ctx, *args)
    ctx.sync()
    assert (from_dev(got) == want).all()


@pytest.mark.parametrize("which", ["scores", "values"])
def test_attention_reports_a_bad_tile_list(ctx, torch_cuda, which):
    from suf_b200 import SufB200Error
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, ATTN[12], 15)
    args, _ = getattr(A, which)()
    for bad in (-1, 3, 2**31 - 1):
        A.layout._tiles[0, 0] = bad
        getattr(at, f"attn_{which}_pair")(ctx, *args)
        with pytest.raises(SufB200Error):
            ctx.sync()
    A.layout._tiles[0, 0] = 0
    A.layout._tiles[0, 1] = 10**9  # a tile past the sequence's last: nothing to do
    getattr(at, f"attn_{which}_pair")(ctx, *args)
    ctx.sync()


@pytest.mark.parametrize("which", ["scores", "values"])
@pytest.mark.parametrize("case", [ATTN[2], ATTN[9]])
def test_attention_reports_bad_pages(ctx, torch_cuda, which, case):
    from suf_b200 import SufB200Error
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, case, 13)
    args, _ = getattr(A, which)()
    call = getattr(at, f"attn_{which}_pair")
    for bad in (-1, A.pages, 2**31 - 1):
        A.layout._table[0, 0] = bad
        call(ctx, *args)
        with pytest.raises(SufB200Error):
            ctx.sync()
        ctx.sync()


def test_layout_refusals(ctx, torch_cuda):
    from suf_b200 import attention as at

    for kw in [dict(q_lens=[1, 2]), dict(ctx_lens=[-1]), dict(q_heads=3), dict(page_size=0), dict(ctx_lens=[33]),
               dict(kv_heads=0)]:
        with pytest.raises(ValueError):
            at.AttnLayout(ctx, **{**dict(q_lens=[1], ctx_lens=[20], block_table=[[0, 1]], page_size=16, q_heads=4,
                                         kv_heads=2), **kw})
    A = _Attn(ctx, torch_cuda, ATTN[2], 1)
    args, _ = A.scores()
    for i, bad in [(0, args[0][:1]), (0, args[0].to(torch_cuda.int32)), (1, args[1][:1]), (2, (args[2][0][1:],) * 2),
                   (3, (1,)), (4, args[4][:, :1]), (5, (args[5][0], args[5][1][:2]))]:
        wrong = list(args)
        wrong[i] = bad
        with pytest.raises(ValueError):
            at.attn_scores_pair(ctx, *wrong)
    with pytest.raises(ValueError):
        at.attn_scores_pair(ctx, *args, out=torch_cuda.empty(3, dtype=torch_cuda.int64, device="cuda"))


def test_attention_on_another_stream_and_in_a_graph(ctx, torch_cuda):
    """Calls on a side stream, and the two products captured in one graph and
    replayed on new inputs, give the words of the eager calls."""
    from suf_b200.attention import attn_scores_pair, attn_values_pair

    torch = torch_cuda
    for case in (ATTN[1], ATTN[12], ATTN[14]):
        A = _Attn(ctx, torch, case, 21)
        (sa, sw), (va, vw) = A.scores(), A.values()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        x, y = attn_scores_pair(ctx, *sa, stream=side), attn_values_pair(ctx, *va, stream=side)
        ctx.sync(side)
        assert (from_dev(x) == sw).all() and (from_dev(y) == vw).all()
        g = torch.cuda.CUDAGraph()
        ox, oy = torch.zeros_like(x), torch.zeros_like(y)
        with torch.cuda.graph(g, stream=side, capture_error_mode="relaxed"):
            attn_scores_pair(ctx, *sa, out=ox, stream=side)
            attn_values_pair(ctx, *va, out=oy, stream=side)
        for _ in range(2):
            (sb, sw), (vb, vw) = A.scores(), A.values()
            sa[0].copy_(sb[0])
            for old, new in zip((*sa[1], *sa[2], *va[0], *va[1], *va[2]), (*sb[1], *sb[2], *vb[0], *vb[1], *vb[2])):
                old.copy_(new)
            g.replay()
            torch.cuda.synchronize()
            ctx.sync()
            assert (from_dev(ox) == sw).all() and (from_dev(oy) == vw).all()


# -- the ragged row max ------------------------------------------------------------------

@pytest.mark.parametrize("lens", [[1], [2], [0, 0], [5, 0, 1, 2, 3, 0], list(range(40)), [129] * 12, [4097, 3, 0, 1000],
                                  [33] * 700, [20000], [1] * 9],
                         ids=lambda x: f"{len(x)}rows-{max(x)}")
def test_rowmax_rounds_match_definition(ctx, torch_cuda, lens):
    from suf_b200 import attention as at

    torch = torch_cuda
    lens = np.asarray(lens)
    rng = np.random.default_rng(int(lens.sum()) + lens.size)
    n = int(lens.sum())
    plan = at.RowMaxPlan(ctx, lens)
    s = [_words(rng, n) for _ in range(2)]
    rows = [np.split(x, np.cumsum(lens)[:-1]) for x in s]
    d_s = cur = tuple(_dev(torch, x) for x in s)
    xh = None
    r = [tuple(int(v) for v in rand_u64(rng, 2)) for _ in range(plan.rounds)]
    if plan.rounds:
        xh = at.rowmax_open_pair(ctx, plan, cur, r[0])
    for k in range(plan.rounds):
        want = np.concatenate([a[0:len(a) - 1:2] - a[1::2] + b[0:len(b) - 1:2] - b[1::2] for a, b in zip(*rows)])
        assert (from_dev(xh) == want + U(r[k][0]) + U(r[k][1])).all()
        relu = [_words(rng, plan.pairs[k]) for _ in range(2)]
        cut = np.cumsum([len(a) // 2 for a in rows[0]])[:-1]
        rows = [[np.concatenate([x[1::2] + q, x[len(x) - len(x) % 2:]]) for x, q in zip(rows[p], np.split(relu[p], cut))]
                for p in (0, 1)]
        cur, xh = at.rowmax_round_pair(ctx, plan, k, cur, tuple(_dev(torch, q) for q in relu),
                                       r[k + 1] if k + 1 < plan.rounds else None)
        for p in (0, 1):
            assert (from_dev(cur[p]) == np.concatenate(rows[p])).all()
    t = at.maxdiff_ragged_pair(ctx, plan, cur, d_s)
    ctx.sync()
    for p in (0, 1):
        top = np.repeat([x[0] if len(x) else U(0) for x in rows[p]], lens).astype(U)
        assert (from_dev(t[p]) == top - s[p]).all()


# -- the block ------------------------------------------------------------------------------

def _model(q, k, v, lens_of, group, f, shift, relu, sm):
    """Plaintext attention of one sequence on reconstructed words: q [n][H][d]
    (already turned), k, v [L][Hkv][d] -> [n][H][d]."""
    from oracle.layer_model import piecewise
    from oracle.softmax_model import softmax_block, tshift

    out = np.zeros_like(q)
    for i in range(q.shape[0]):
        for h in range(q.shape[1]):
            m = lens_of(i)
            if m == 0:
                continue
            s = tshift(k[:m, h // group] @ q[i, h], f + shift)
            c = s.copy()
            while c.size > 1:  # the tournament on a row of any length
                odd = c[c.size - c.size % 2:]
                c = np.concatenate([c[1::2] + piecewise(relu, c[0:c.size - 1:2] - c[1::2]), odd])
            p = softmax_block(c[0] - s, np.array([0, m]), sm)
            out[i, h] = tshift(p @ v[:m, h // group], f)
    return out


def test_block_prompt_then_single_tokens_matches_model(ctx, torch_cuda):
    """A prompt of three packed sequences and then two decode steps over the
    same cache, every step exact in Z_2^64: the reconstructed output equals the
    plaintext model word for word."""
    from oracle.layer_model import load_layer_tables
    from oracle.softmax_model import load_tables
    from suf_b200.attention import AttnLayout, CachedAttentionPair, ShareCache, rope_tables

    torch = torch_cuda
    f, hq, hkv, dh, page = 12, 4, 2, 64, 8
    rng = np.random.default_rng(9)
    relu, sm = load_layer_tables()["relu"], load_tables()
    cache = ShareCache(ctx, 16, hkv, dh, page, seed=3)
    rope = rope_tables(ctx, 256, 32, f)
    hc, hs = (t.cpu().numpy().astype(np.int64) for t in rope)
    order = rng.permutation(16)
    have = [np.zeros((0, hkv, dh), dtype=U) for _ in range(3)]
    vals = [np.zeros((0, hkv, dh), dtype=U) for _ in range(3)]
    tables = [order[0:5].tolist(), order[5:9].tolist(), order[9:14].tolist()]
    for step, new in enumerate([[19, 1, 30], [1, 1, 1], [1, 0, 2]]):
        q_lens = new
        ctx_lens = [have[b].shape[0] + new[b] for b in range(3)]
        layout = AttnLayout(ctx, q_lens, ctx_lens, tables, page, hq, hkv)
        blk = CachedAttentionPair(ctx, cache, layout, seed=50 + step, rope=rope)
        T = layout.tokens
        x = np.rint(rng.normal(0.0, 1.0, (T, (hq + 2 * hkv), dh)) * 2**f).astype(np.int64)
        s0 = _words(rng, T, hq + 2 * hkv, dh)
        sh = [_dev(torch, s0), _dev(torch, x.view(U) - s0)]
        pos = np.concatenate([np.arange(have[b].shape[0], ctx_lens[b]) for b in range(3)]).astype(np.int32)
        slots = np.concatenate([[tables[b][j // page] * page + j % page for j in range(have[b].shape[0], ctx_lens[b])]
                                for b in range(3)]).astype(np.int64)
        o = blk.run(tuple(s[:, :hq] for s in sh), tuple(s[:, hq:hq + hkv] for s in sh),
                    tuple(s[:, hq + hkv:] for s in sh), torch.from_numpy(pos).cuda(), torch.from_numpy(slots).cuda())
        ctx.sync()
        got = from_dev(o[0]) + from_dev(o[1])
        t0 = 0
        for b in range(3):
            n, L = q_lens[b], ctx_lens[b]
            turned = np.stack([_turn(x[t0 + i, :hq + hkv], hc[pos[t0 + i]], hs[pos[t0 + i]], 32, f, False)
                               for i in range(n)]).view(U) if n else np.zeros((0, hq + hkv, dh), dtype=U)
            have[b] = np.concatenate([have[b], turned[:, hq:]])
            vals[b] = np.concatenate([vals[b], x[t0:t0 + n, hq + hkv:].view(U)])
            want = _model(turned[:, :hq], have[b], vals[b], lambda i: L - n + i + 1, hq // hkv, f, 3, relu, sm)
            assert (got[t0:t0 + n] == want).all(), (step, b)
            t0 += n


def test_block_runs_on_a_side_stream_and_in_a_graph(ctx, torch_cuda):
    """A decode step captured once and replayed on new shares gives the words
    of the eager call on the same material."""
    from suf_b200.attention import AttnLayout, CachedAttentionPair, ShareCache, rope_tables

    torch = torch_cuda
    rng = np.random.default_rng(4)
    hq, hkv, dim, page = 4, 2, 64, 8
    cache = ShareCache(ctx, 8, hkv, dim, page, seed=5)
    layout = AttnLayout(ctx, [3, 1], [19, 30], [[0, 2, 4], [1, 3, 5, 7]], page, hq, hkv)
    blk = CachedAttentionPair(ctx, cache, layout, seed=6, rope=rope_tables(ctx, 64, dim, 12), interleaved=True)
    pos = torch.tensor([16, 17, 18, 29], dtype=torch.int32, device="cuda")
    slots = torch.tensor([4 * 8 + 0, 4 * 8 + 1, 4 * 8 + 2, 7 * 8 + 5], dtype=torch.int64, device="cuda")
    cache.ek.copy_(-cache.bk[0] - cache.bk[1] + 4096)  # cached keys and values of one
    cache.ev.copy_(-cache.bv[0] - cache.bv[1] + 4096)

    def shares():
        x = np.rint(rng.normal(0.0, 1.0, (4, hq + 2 * hkv, dim)) * 4096).astype(np.int64)
        s0 = _words(rng, *x.shape)
        return [_dev(torch, s0), _dev(torch, x.view(U) - s0)]

    buf = shares()
    q, k, v = (tuple(b[:, i:j] for b in buf) for i, j in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    blk.run(q, k, v, pos, slots, stream=side)  # warm-up outside the capture
    ctx.sync(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side, capture_error_mode="relaxed"):
        o = blk.run(q, k, v, pos, slots, stream=side)
    for _ in range(2):
        for b, n in zip(buf, shares()):
            b.copy_(n)
        g.replay()
        torch.cuda.synchronize()
        ctx.sync()
        e = blk.run(q, k, v, pos, slots)
        ctx.sync()
        assert all((from_dev(x) == from_dev(y)).all() for x, y in zip(o, e))


def test_block_without_new_tokens(ctx, torch_cuda):
    from suf_b200.attention import AttnLayout, CachedAttentionPair, ShareCache

    cache = ShareCache(ctx, 4, 2, 64, 8, seed=1)
    blk = CachedAttentionPair(ctx, cache, AttnLayout(ctx, [0, 0], [9, 0], [[0, 1], []], 8, 4, 2), seed=2)
    none = tuple(torch_cuda.zeros((0, n, 64), dtype=torch_cuda.int64, device="cuda") for n in (4, 2, 2))
    o = blk.run(*((x, x) for x in none), None, torch_cuda.zeros(0, dtype=torch_cuda.int64, device="cuda"))
    ctx.sync()
    assert o[0].shape == (0, 4, 64)


def test_truncation_pair_with_and_without_queries(ctx, torch_cuda):
    from suf_b200.attention import TruncPair

    torch = torch_cuda
    rng = np.random.default_rng(8)
    x = rng.integers(-(2**61), 2**61, 5000, dtype=np.int64)
    bare = next(s for s in range(200) if int(TruncPair(ctx, 1, seed=s).desc[0].nq) == 0)
    for f, seed in ((12, 3), (16, 4), (1, bare)):
        tr = TruncPair(ctx, f, seed=seed)
        xh = _dev(torch, x.view(U) + U(tr.r[0]) + U(tr.r[1]))
        y = torch.empty_like(xh), torch.empty_like(xh)
        tr.eval_pair(ctx, xh, *y)
        ctx.sync()
        assert ((from_dev(y[0]) + from_dev(y[1])).view(np.int64) == x >> f).all()


def test_products_are_exact_at_full_depth(ctx, torch_cuda):
    """Every operand word all ones: the largest sums the int32 diagonals of the
    tensor-core path can meet, over 4,096 keys (the exact depth) and 5,000."""
    from suf_b200.attention import AttnLayout, attn_scores_pair, attn_values_pair

    torch = torch_cuda
    n, dh, page = 64, 128, 64
    for L in (4096, 5000):
        pages = -(-L // page)
        lay = AttnLayout(ctx, [n], [L], [list(range(pages))], page, 1, 1, causal=False)
        ones = torch.full((pages, 1, page, dh), -1, dtype=torch.int64, device="cuda")
        zero = torch.zeros_like(ones)
        pool = (ones, (ones, zero))  # E and W all ones
        z_q, z_p = torch.zeros((n, 1, dh), dtype=torch.int64, device="cuda"), torch.zeros(n * L, dtype=torch.int64,
                                                                                         device="cuda")
        out = attn_values_pair(ctx, (z_p - 1, z_p), (z_p, z_p), (z_q, z_q), (0, 0), *pool, lay)
        ctx.sync()
        assert (from_dev(out) == U(2 * L)).all()  # (-1)(-1) twice per key
        out = attn_scores_pair(ctx, z_q - 1, (z_q, z_q), (z_p, z_p), (0, 0), *pool, lay)
        ctx.sync()
        assert (from_dev(out) == U(2 * dh)).all()


def test_pages_past_32_bit_offsets(ctx, torch_cuda):
    """Pages whose words lie past 2^32 in the pool (one pool stands for the
    opened words and both masks: it is only read)."""
    from suf_b200.attention import AttnLayout, attn_scores_pair, attn_values_pair

    torch = torch_cuda
    hkv, dh, page = 8, 128, 64
    words = hkv * dh * page
    pages = 2**32 // words + 4
    if torch.cuda.mem_get_info()[0] < 8 * words * pages + 2**31:
        pytest.skip("needs 37 GB of free device memory")
    pool = torch.empty((pages, hkv, page, dh), dtype=torch.int64, device="cuda")
    rng = np.random.default_rng(1)
    ids = [pages - 1, 3, pages - 3]
    small = _words(rng, 3, hkv, page, dh)
    for i, p in enumerate(ids):
        pool[p] = _dev(torch, small[i])
    for n in (1, 12):  # row kernels, tensor cores
        L = 150
        lay = AttnLayout(ctx, [n], [L], [ids], page, hkv, hkv)
        lens = [L - n + i + 1 for i in range(n)]
        k = small.transpose(1, 0, 2, 3).reshape(hkv, -1, dh)[:, :L]
        d, c = _words(rng, n, hkv, dh), _words(rng, hkv * sum(lens))
        z_q, z_p = np.zeros_like(d), np.zeros_like(c)
        dz_q, dz_p = _dev(torch, z_q), _dev(torch, z_p)
        got = attn_scores_pair(ctx, _dev(torch, d), (dz_q, dz_q), (_dev(torch, c), dz_p), (0, 0), pool, (pool, pool), lay)
        ctx.sync()
        want = np.concatenate([U(3) * (k[h, :lens[i]] @ d[i, h]) for h in range(hkv) for i in range(n)]) + c
        assert (from_dev(got) == want).all()
        got = attn_values_pair(ctx, (_dev(torch, c), dz_p), (dz_p, dz_p), (dz_q, dz_q), (0, 0), pool, (pool, pool), lay)
        ctx.sync()
        want, at = np.zeros_like(d), 0
        for h in range(hkv):
            for i in range(n):
                want[i, h] = U(3) * (c[at:at + lens[i]] @ k[h, :lens[i]])
                at += lens[i]
        assert (from_dev(got) == want).all()
    del pool
    torch.cuda.empty_cache()


def _many_sequences(prompts):
    """A batch whose search for a block's sequence takes several steps: empty
    caches, runs of every length, one long cache, with `prompts` whole prompts
    between the single tokens."""
    rng = np.random.default_rng(31)
    seqs = [(1, int(L)) for L in rng.choice([0, 1, 2, 31, 63, 64, 65, 127, 200, 257], 1100)]
    seqs[700] = (1, 1500)
    seqs[3] = seqs[40] = (0, 90)
    if prompts:
        for i in (0, 33, 500, 1099):
            seqs[i] = (12, 80 + i % 7)
    return (seqs, 2, 1, 6, 16, True)


@pytest.mark.parametrize("which", ["scores", "values"])
@pytest.mark.parametrize("prompts", [False, True])
def test_many_sequences_match_definition(ctx, torch_cuda, which, prompts):
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, _many_sequences(prompts), 33)
    args, want = getattr(A, which)()
    got = getattr(at, f"attn_{which}_pair")(ctx, *args)
    ctx.sync()
    assert (from_dev(got) == want).all()


@pytest.mark.parametrize("which", ["scores", "values"])
@pytest.mark.parametrize("case", [ATTN[3], ATTN[12], ATTN[14]])
def test_attention_reports_bad_lengths(ctx, torch_cuda, which, case):
    """Cached lengths that fall, or pass what the host was told: reported, also
    where no block's search finds the sequence."""
    from suf_b200 import SufB200Error
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, case, 34)
    args, want = getattr(A, which)()
    call, good = getattr(at, f"attn_{which}_pair"), A.layout._ctx.clone()
    for at_, bad in [(-1, 0), (1, -5), (1, 2**31 - 1), (-1, 2**31 - 1)]:
        A.layout._ctx[at_] = bad
        call(ctx, *args)
        with pytest.raises(SufB200Error):
            ctx.sync()
        A.layout._ctx.copy_(good)
    got = call(ctx, *args)
    ctx.sync()
    assert (from_dev(got) == want).all()


@pytest.mark.parametrize("case", [([(70, 150), (33, 20)], 4, 2, 134, 16, True), ([(150, 300), (0, 3)], 2, 1, 256, 64, True),
                                  ([(20, 5), (1, 40)], 3, 1, 130, 7, True), ([(24, 131)], 2, 2, 224, 32, False)])
def test_scores_of_wide_heads_in_two_parts(ctx, torch_cuda, case):
    """Heads above 128 words: the second part adds to the first one's words, and
    leaves what is behind the last row alone."""
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, case, 35)
    args, want = A.scores()
    buf, out = _guarded(torch_cuda, want)
    at.attn_scores_pair(ctx, *args, out=out)
    ctx.sync()
    assert (from_dev(out) == want).all() and (buf[want.size:] == 77).all()


def test_two_streams_and_two_graphs_at_once(ctx, torch_cuda):
    """Calls in flight on two streams, and two captured graphs replayed beside
    one another, share no workspace: every result as if alone."""
    from suf_b200 import attention as at

    torch = torch_cuda
    jobs = []
    for i, case in enumerate([([(600, 900), (1, 700)], 8, 2, 64, 64, True), ([(300, 1000)], 4, 2, 160, 16, True)]):
        A = _Attn(ctx, torch, case, 40 + i)
        for which in ("scores", "values"):
            call, (args, _) = getattr(at, f"attn_{which}_pair"), getattr(A, which)()
            jobs.append((A, call, args, call(ctx, *args)))
    ctx.sync()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        outs = [torch.empty_like(want) for *_, want in jobs]
        torch.cuda.synchronize()
        for st, out, (_, call, args, _) in zip(streams, outs, jobs):
            call(ctx, *args, out=out, stream=st)
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out, (*_, want) in zip(outs, jobs))
    graphs = []
    for st, out, (_, call, args, _) in zip(streams, outs, jobs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            call(ctx, *args, out=out, stream=st)
        graphs.append(g)
    for _ in range(3):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out, (*_, want) in zip(outs, jobs))
    ctx.sync()


@pytest.mark.parametrize("which", ["scores", "values"])
def test_a_workspace_that_cannot_be_had_is_this_calls_error_only(ctx, torch_cuda, which):
    """More cached tokens than any memory holds planes for: refused by the
    allocator, and the calls after it work."""
    from suf_b200 import SufB200Error
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, ([(20, 40)], 64, 64, 2, 16, True), 50)
    args, want = getattr(A, which)()
    call, cached = getattr(at, f"attn_{which}_pair"), A.layout._seqs.cached
    A.layout._seqs.cached = 2**30  # terabytes of planes
    with pytest.raises(SufB200Error):
        call(ctx, *args)
    A.layout._seqs.cached = cached
    got = call(ctx, *args)
    ctx.sync()
    assert (from_dev(got) == want).all()
