"""The forms of the tensor-core products that whole prompts take, against the
definition in 64-bit words (tolerance zero): several key tiles a CTA, whole
rows of values of more than eight chunks, ranges cut at the exact depth, and
short sequences beside them.  Which form a case takes follows from the launch
rule restated here, and every case says which one it is for.  Then workspaces and
bounds of mixed batches, appends and row maxima past one grid, and the block's
rows with one key or none."""
from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import from_dev, rand_u64, to_dev
from tests.test_gpu_attention import GUARD, U, _Attn, _guarded, _model, _rope_case, test_rowmax_rounds_match_definition as _rowmax

pytestmark = pytest.mark.gpu


def _ceil(a, b):
    return -(-a // b)


def _launch(ctx, A):
    """(key tiles per CTA of the scores, keys per CTA of the values, longest
    context) of the sequences with more than eight rows per key head."""
    group = A.hq // A.hkv
    long_ = [(n, L) for n, L in zip(A.q, A.L) if n * group > 8]
    tiles, ctx_len = sum(_ceil(n * group, 64) for n, _ in long_), max(L for _, L in long_)
    two = 2 * ctx.sm_count
    nt, nch = _ceil(ctx_len, 128), _ceil(ctx_len, 32)
    span = min(_ceil(nt * tiles * A.hkv, two), nt)
    units = tiles * _ceil(A.dh, 128) * A.hkv
    keys = min(nch if units > ctx.sm_count else max(8, _ceil(units * nch, two)), nch) * 32
    return span, min(keys, 4096), ctx_len


SCORES = [  # (case, least key tiles a CTA); the last tile and the last row tile are ragged
    (([(200, 1290)], 16, 16, 16, 64, True), 3),
    (([(128, 2000), (1, 300)], 32, 32, 8, 32, True), 4),
    (([(77, 1500), (130, 140)], 40, 20, 34, 16, False), 2),
    (([(100, 1100)], 24, 24, 130, 64, True), 2),  # a wide head: both parts walk several tiles
    (([(60, 50), (90, 1000), (3, 700)], 60, 20, 40, 100, True), 2),
]


@pytest.mark.parametrize("case,least", SCORES)
def test_scores_of_several_key_tiles_a_cta(ctx, torch_cuda, case, least):
    from suf_b200.attention import attn_scores_pair

    A = _Attn(ctx, torch_cuda, case, 61)
    assert _launch(ctx, A)[0] >= least
    args, want = A.scores()
    buf, out = _guarded(torch_cuda, want)
    for _ in range(2):
        out.fill_(5)
        attn_scores_pair(ctx, *args, out=out)
        ctx.sync()
        assert (from_dev(out) == want).all() and (buf[want.size:] == 77).all()


VALUES = [  # (case, whole rows)
    (([(256, 600)], 40, 40, 8, 64, True), True),
    (([(256, 600), (1, 400), (2, 300)], 40, 40, 8, 64, True), True),  # the short ones start from C, the prompt does not
    (([(1, 290), (70, 400), (0, 33), (64, 333)], 60, 60, 18, 16, False), True),
    (([(40, 30), (100, 400), (1, 380)], 40, 20, 130, 32, True), True),  # two tiles of words, queries without keys
    (([(12, 5000)], 150, 150, 2, 64, True), False),  # whole rows would pass the exact depth
    (([(16, 4500), (1, 4200)], 160, 160, 2, 64, False), False),
    (([(70, 3000), (1, 700)], 16, 16, 24, 64, True), False),  # ranges of more than eight chunks
]


@pytest.mark.parametrize("case,whole", VALUES)
def test_values_of_whole_rows_and_of_ranges(ctx, torch_cuda, case, whole):
    from suf_b200.attention import attn_values_pair

    A = _Attn(ctx, torch_cuda, case, 62)
    _, keys, longest = _launch(ctx, A)
    assert (keys >= longest) == whole and keys > 256
    args, want = A.values()
    buf, out = _guarded(torch_cuda, want)
    for _ in range(2):
        out.fill_(5)
        attn_values_pair(ctx, *args, out=out)
        ctx.sync()
        assert (from_dev(out) == want).all() and (buf[want.size:] == 77).all()


@pytest.mark.parametrize("L,keys", [(4096, 4096), (5000, 4096)])
def test_values_are_exact_over_4096_keys_a_cta(ctx, torch_cuda, L, keys):
    """Every word all ones, and more row tiles than SMs, so that one CTA adds up
    4,096 keys: 8,192 products of 255 x 255 on every limb pair, eight pairs on the
    highest diagonal, 8 * 8,192 * 255^2 = 4,261,478,400 < 2^32."""
    from suf_b200.attention import AttnLayout, attn_values_pair

    torch = torch_cuda
    n, h, dh, page = 12, ctx.sm_count + 2, 32, 64
    pages = _ceil(L, page)
    lay = AttnLayout(ctx, [n], [L], [list(range(pages))], page, h, h, causal=False)
    units, nch = h, _ceil(L, 32)
    assert units > ctx.sm_count and min(nch * 32, 4096) == keys
    ones = torch.full((pages, h, page, dh), -1, dtype=torch.int64, device="cuda")
    pool = (ones, (ones, torch.zeros_like(ones)))  # E and W all ones
    z_p = torch.zeros(lay.packed, dtype=torch.int64, device="cuda")
    z_q = torch.zeros((n, h, dh), dtype=torch.int64, device="cuda")
    buf = torch.full((z_q.numel() + GUARD,), 77, dtype=torch.int64, device="cuda")
    out = buf[:z_q.numel()].view(z_q.shape)
    attn_values_pair(ctx, (z_p - 1, z_p), (z_p, z_p), (z_q, z_q), (0, 0), *pool, lay, out=out)
    ctx.sync()
    assert (from_dev(out) == U(2 * L)).all() and (buf[z_q.numel():] == 77).all()  # (-1)(-1) twice per key


@pytest.mark.parametrize("which", ["scores", "values"])
def test_workspace_follows_the_prompts_and_not_the_batch(ctx, torch_cuda, which):
    """A prompt of 40 tokens beside 300 idle caches of 2^22 tokens (all on the same
    pages: nothing reads them): planes of all of them would take 640 GB."""
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, ([(20, 40)], 2, 2, 2, 65536, True), 63)
    args, want = getattr(A, which)()
    idle = [A.table[0] * 64] * 300
    lay = at.AttnLayout(ctx, A.q + [0] * 300, A.L + [2**22] * 300, A.table + idle, A.page, A.hq, A.hkv)
    got = getattr(at, f"attn_{which}_pair")(ctx, *args[:-1], lay)
    ctx.sync()
    assert (from_dev(got) == want).all()


MIXED = [  # long sequences between short ones, idle ones and empty caches
    ([(1, 300), (70, 130), (0, 200), (1, 0), (33, 257), (2, 77), (20, 5)], 4, 2, 66, 16, True),
    ([(12, 0), (1, 500), (1, 129)], 2, 1, 32, 64, True),  # the long sequence has no keys: nothing takes room
    ([(1, 40), (24, 300), (1, 128), (130, 128)], 3, 1, 160, 32, False),
]


@pytest.mark.parametrize("which", ["scores", "values"])
@pytest.mark.parametrize("case", MIXED)
def test_long_and_short_sequences_with_and_without_places(ctx, torch_cuda, which, case):
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, case, 64)
    args, want = getattr(A, which)()
    call = getattr(at, f"attn_{which}_pair")
    assert A.layout._seqs.plane_keys > 0
    for places in (True, False):
        if not places:
            A.layout._seqs.d_plane_keys, A.layout._seqs.plane_keys = None, 0
        buf, out = _guarded(torch_cuda, want)
        call(ctx, *args, out=out)
        ctx.sync()
        assert (from_dev(out) == want).all() and (buf[want.size:] == 77).all()


@pytest.mark.parametrize("which", ["scores", "values"])
def test_attention_reports_bad_places(ctx, torch_cuda, which):
    from suf_b200 import SufB200Error
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, MIXED[0], 65)
    args, want = getattr(A, which)()
    call, good = getattr(at, f"attn_{which}_pair"), A.layout._places.clone()
    for i, bad in [(1, -128), (1, 64), (2, 128), (5, 2**31 - 1), (4, 2**31 - 128), (4, -2**31)]:
        A.layout._places[i] = bad
        call(ctx, *args)
        with pytest.raises(SufB200Error):
            ctx.sync()
        A.layout._places.copy_(good)
    got = call(ctx, *args)
    ctx.sync()
    assert (from_dev(got) == want).all()


BESIDE = [  # a short sequence whose cache is longer than the prompts': theirs alone decide how they are split
    (([(200, 1290), (1, 4000)], 16, 16, 16, 64, True), 3),
    (([(256, 600), (1, 3000), (4, 700)], 40, 40, 8, 64, True), 3),   # whole rows of values
    (([(1, 5000), (60, 90), (2, 3), (90, 1000)], 60, 20, 40, 100, True), 2),
    (([(1, 2000), (40, 300), (1, 65)], 8, 2, 130, 16, False), 1),    # groups of four: four rows beside a prompt
]


@pytest.mark.parametrize("which", ["scores", "values"])
@pytest.mark.parametrize("case,span", BESIDE)
def test_prompts_beside_longer_caches(ctx, torch_cuda, which, case, span):
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, case, 66)
    assert _launch(ctx, A)[0] >= span and _launch(ctx, A)[2] == A.layout._seqs.long_ctx < max(A.L)
    args, want = getattr(A, which)()
    call = getattr(at, f"attn_{which}_pair")
    for given in (True, False):  # without the bounds: the batch's longest context, eight rows
        if not given:
            A.layout._seqs.long_ctx = A.layout._seqs.short_rows = 0
        buf, out = _guarded(torch_cuda, want)
        call(ctx, *args, out=out)
        ctx.sync()
        assert (from_dev(out) == want).all() and (buf[want.size:] == 77).all()


@pytest.mark.parametrize("which", ["scores", "values"])
def test_attention_reports_sequences_past_their_bounds(ctx, torch_cuda, which):
    from suf_b200 import SufB200Error
    from suf_b200 import attention as at

    A = _Attn(ctx, torch_cuda, BESIDE[3][0], 67)
    args, _ = getattr(A, which)()
    call, s = getattr(at, f"attn_{which}_pair"), A.layout._seqs
    for kw in (dict(long_ctx=299), dict(short_rows=3)):
        old = {k: getattr(s, k) for k in kw}
        for k, v in kw.items():
            setattr(s, k, v)
        call(ctx, *args)
        with pytest.raises(SufB200Error):
            ctx.sync()
        for k, v in old.items():
            setattr(s, k, v)
    call(ctx, *args)
    ctx.sync()


def test_one_token_of_views_with_different_strides(ctx, torch_cuda):
    """The parties' shares of one token, one in a fused row and one by itself."""
    from suf_b200.attention import rope_append_pair

    for case in [(1, 12, 4, 64, 64, False, 64, 12, 40, 0), (1, 3, 1, 18, 6, True, 3, 15, 40, 0)]:
        args, kw, want, got, _ = _rope_case(ctx, torch_cuda, case, seed=9)
        q, k, v = ((x, y.clone(memory_format=torch_cuda.contiguous_format)) for x, y in args[:3])
        assert q[0].stride() != q[1].stride()
        rope_append_pair(ctx, q, k, v, *args[3:], **kw)
        ctx.sync()
        assert all((from_dev(g) == w).all() for w, g in zip(want, got))


def test_a_page_written_again_under_fresh_masks(ctx, torch_cuda):
    """The same rows appended twice into one page: under fresh masks the two
    openings share no word, and each opens to the rows."""
    from suf_b200.attention import ShareCache, rope_append_pair

    torch = torch_cuda
    cache = ShareCache(ctx, 3, 2, 16, 8, seed=4)
    x = [torch.randint(-(2**63), 2**63 - 1, (8, 2, 16), dtype=torch.int64, device="cuda") for _ in range(4)]
    slots = torch.arange(8, 16, dtype=torch.int64, device="cuda")
    opened = []
    for _ in range(2):
        rope_append_pair(ctx, None, (x[0], x[1]), (x[2], x[3]), None, slots, None, None, None, None, cache)
        ctx.sync()
        opened.append((cache.ek[1].clone(), cache.ev[1].clone()))
        for e, b, s in ((cache.ek, cache.bk, x[:2]), (cache.ev, cache.bv, x[2:])):
            assert torch.equal((e[1] + b[0][1] + b[1][1]).transpose(0, 1), s[0] + s[1])
        cache.fresh_masks([1])
    assert (opened[0][0] != opened[1][0]).all() and (opened[0][1] != opened[1][1]).all()


@pytest.mark.parametrize("new", [[(1, 1)], [(1, 1), (1, 1), (1, 1)], [(5, 3), (1, 1)], [(9, 2), (1, 12), (4, 1)], [(3, 0), (2, 2)]])
def test_block_with_single_keys_and_rows_that_see_nothing(ctx, torch_cuda, new):
    """First tokens (one key: no row max round) and queries in front of what is
    cached (empty rows through the row max and the softmax block), against the
    plaintext model word for word; an empty row gives zero."""
    from oracle.layer_model import load_layer_tables
    from oracle.softmax_model import load_tables
    from suf_b200.attention import AttnLayout, CachedAttentionPair, ShareCache

    torch = torch_cuda
    hq, hkv, dh, page = 4, 2, 16, 4
    rng = np.random.default_rng(17)
    cache = ShareCache(ctx, 16, hkv, dh, page, seed=8)
    q_lens, ctx_lens = [n for n, _ in new], [L for _, L in new]
    tables = [[3 * b + j for j in range(3)] for b in range(len(new))]
    blk = CachedAttentionPair(ctx, cache, AttnLayout(ctx, q_lens, ctx_lens, tables, page, hq, hkv), seed=19)
    T = sum(q_lens)
    x = np.rint(rng.normal(0.0, 1.0, (T, hq + 2 * hkv, dh)) * 4096).astype(np.int64)
    old = [np.rint(rng.normal(0.0, 1.0, (2, max(L - n, 0), hkv, dh)) * 4096).astype(np.int64) for n, L in new]
    slots, t0, spare = [], 0, 12 * page
    for b, (n, L) in enumerate(new):
        for j in range(max(L - n, 0)):  # what was cached before
            pg, at = tables[b][j // page], j % page
            for pool, m, y in ((cache.ek, cache.bk, old[b][0]), (cache.ev, cache.bv, old[b][1])):
                pool[pg, :, at] = torch.from_numpy(y[j]).cuda() - m[0][pg, :, at] - m[1][pg, :, at]
        for i in range(n):
            j = L - n + i
            slots.append(tables[b][j // page] * page + j % page if j >= 0 else spare)
            spare += j < 0
    s0 = rand_u64(rng, x.size).reshape(x.shape)
    sh = [to_dev(torch, s0), to_dev(torch, x.view(U) - s0)]
    o = blk.run(tuple(s[:, :hq] for s in sh), tuple(s[:, hq:hq + hkv] for s in sh), tuple(s[:, hq + hkv:] for s in sh),
                None, torch.tensor(slots, dtype=torch.int64, device="cuda"))
    ctx.sync()
    got = from_dev(o[0]) + from_dev(o[1])
    relu, sm = load_layer_tables()["relu"], load_tables()
    for b, (n, L) in enumerate(new):
        k, v = (np.concatenate([old[b][w], x[t0 + max(n - L, 0):t0 + n, hq + w * hkv:hq + (w + 1) * hkv]]).view(U)
                for w in (0, 1))
        assert len(k) == L
        want = _model(x[t0:t0 + n, :hq].view(U), k, v, lambda i: max(0, L - n + i + 1), hq // hkv, 12, 2, relu, sm)
        assert (got[t0:t0 + n] == want).all(), b
        t0 += n


def test_append_of_a_prompt_on_a_side_stream_and_in_a_graph(ctx, torch_cuda):
    """Enough turned words for the packed carries: their table is the call's own,
    also where two captured appends replay beside one another."""
    from suf_b200.attention import rope_append_pair

    torch = torch_cuda
    jobs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for inter, st in zip((False, True), streams):
        args, kw, want, got, _ = _rope_case(ctx, torch, (300, 32, 8, 128, 128, inter, 64, 12, 44, 2), 70 + inter)
        before = [g.clone() for g in got]
        torch.cuda.synchronize()
        rope_append_pair(ctx, *args, **kw, stream=st)
        ctx.sync(st)
        assert all((from_dev(g) == w).all() for w, g in zip(want, got))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st, capture_error_mode="relaxed"):
            rope_append_pair(ctx, *args, **kw, stream=st)
        jobs.append((graph, st, before, want, got, args))
    for _ in range(3):
        for _, _, before, _, got, _ in jobs:
            for g, b in zip(got, before):
                g.copy_(b)
        torch.cuda.synchronize()
        for graph, st, *_ in jobs:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        ctx.sync()
        for _, _, _, want, got, _ in jobs:
            assert all((from_dev(g) == w).all() for w, g in zip(want, got))


def test_append_of_more_rows_than_the_grid_has_warps(ctx, torch_cuda):
    """100,000 tokens of 96 heads: 9.6 million rows on 2^20 blocks of eight."""
    from suf_b200.attention import ShareCache, TruncPair, rope_append_pair, rope_tables

    torch = torch_cuda
    T, hq, hkv, dh, page, f = 100_000, 60, 18, 2, 64, 12
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randint(-(2**40), 2**40, (T, hq + 2 * hkv, dh), dtype=torch.int64, device="cuda", generator=g)
    s = torch.randint(-(2**63), 2**63 - 1, x.shape, dtype=torch.int64, device="cuda", generator=g)
    sh = (s, x - s)
    q, k, v = (tuple(t[:, i:j] for t in sh) for i, j in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    cache = ShareCache(ctx, -(-T // page), hkv, dh, page, seed=5)
    slots = torch.randperm(cache.pages * page, device="cuda", generator=g)[:T]
    pos = torch.randint(0, 4096, (T,), device="cuda", generator=g).to(torch.int32)
    cos, sin = rope_tables(ctx, 4096, dh, f)
    a = tuple(torch.randint(-(2**63), 2**63 - 1, (T, hq, dh), dtype=torch.int64, device="cuda", generator=g) for _ in range(2))
    d_q = rope_append_pair(ctx, q, k, v, pos, slots, cos, sin, TruncPair(ctx, f, seed=6), a, cache)
    ctx.sync()
    c, n = (t[pos.long(), 0].long()[:, None] for t in (cos, sin))
    y = x.clone()
    y[:, :hq + hkv, 0] = (x[:, :hq + hkv, 0] * c - x[:, :hq + hkv, 1] * n) >> f
    y[:, :hq + hkv, 1] = (x[:, :hq + hkv, 1] * c + x[:, :hq + hkv, 0] * n) >> f
    assert torch.equal(d_q, y[:, :hq] - a[0] - a[1])
    for e, b, rows in ((cache.ek, cache.bk, y[:, hq:hq + hkv]), (cache.ev, cache.bv, y[:, hq + hkv:])):
        assert torch.equal((e + b[0] + b[1]).transpose(1, 2).reshape(-1, hkv, dh)[slots], rows)


@pytest.mark.parametrize("rows,most", [(100_000, 9), (20_000, 40), (3_000, 900)])
def test_rowmax_of_more_rows_than_the_grid_takes_at_once(ctx, torch_cuda, rows, most):
    rng = np.random.default_rng(rows)
    _rowmax(ctx, torch_cuda, rng.integers(0, most + 1, rows).tolist())
