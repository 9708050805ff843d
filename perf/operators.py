"""Cases for the operators of attention over a paged cache of secret-shared
keys and values (both parties' shares on one GPU, Z_2^64, f = 12 fractional
bits): the rotary append, the attention scores, the attention values and the
row max over ragged rows.

With `own` false, run() computes them from elementary torch operations; with
`own` true it makes the calls of suf_b200.attention.  Every output is an
opened (public) value or a share, whole words mod 2^64.
"""
import math

import numpy as np
import torch

own = False

F = 12  # fractional bits of every value, cosine and sine
# a decode batch: "new tokens / cached tokens, the new ones included" of every sequence
LONG = "1/16384 1/12001 1/1 1/9000 1/16001 1/4097 1/15000 1/777"
_CTX = []


def _ctx():
    """The engine context a program keeps for its lifetime."""
    if not _CTX:
        from suf_b200.engine import Context, host_mt19937_64

        c = Context(0)
        c.prg_init(host_mt19937_64(0x5EED_0001, 16).view(np.uint8))
        _CTX.append(c)
    return _CTX[0]


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one new token of one client, 12 heads of 64: the launch latency of a decode step
        {"name": "rope 1 token 12x64", "op": "rope", "tokens": 1, "hq": 12, "hkv": 12, "dh": 64, "rot": 64,
         "interleaved": False, "page": 64, "max_pos": 2048, "pad": 0},
        # a decode batch with grouped heads, half of each head rotated, interleaved pairs, long positions, padding rows
        {"name": "rope 77 tokens 32/8x128 part", "op": "rope", "tokens": 77, "hq": 32, "hkv": 8, "dh": 128, "rot": 64,
         "interleaved": True, "page": 32, "max_pos": 131072, "pad": 13},
        # a packed prompt of odd length appended at once
        {"name": "rope 4133 tokens 32/8x128", "op": "rope", "tokens": 4133, "hq": 32, "hkv": 8, "dh": 128, "rot": 128,
         "interleaved": False, "page": 64, "max_pos": 8192, "pad": 0},
        # one token against a short cache, 12 heads of 64
        {"name": "scores 1 token ctx 129", "op": "scores", "seqs": "1/129", "hq": 12, "hkv": 12, "dh": 64,
         "page": 64, "causal": True},
        # a decode batch over long caches of very different lengths, grouped heads
        {"name": "scores decode long 32/8x128", "op": "scores", "seqs": LONG, "hq": 32, "hkv": 8,
         "dh": 128, "page": 64, "causal": True},
        # the whole-prompt square of the 12-head layer, no causal mask
        {"name": "scores square 128 12x64", "op": "scores", "seqs": "128/128", "hq": 12, "hkv": 12, "dh": 64,
         "page": 64, "causal": False},
        # packed prompts: a fresh one, one continued behind a cached prefix, one single token
        {"name": "scores prompt 16/4x128", "op": "scores", "seqs": "2048/2048 700/1724 1/33", "hq": 16,
         "hkv": 4, "dh": 128, "page": 64, "causal": True},
        # the value products of the same three kinds of step
        {"name": "values 1 token ctx 129", "op": "values", "seqs": "1/129", "hq": 12, "hkv": 12, "dh": 64,
         "page": 64, "causal": True},
        {"name": "values decode long 32/8x128", "op": "values", "seqs": LONG, "hq": 32, "hkv": 8,
         "dh": 128, "page": 64, "causal": True},
        {"name": "values prompt 16/4x128", "op": "values", "seqs": "2048/2048 700/1724 1/33", "hq": 16,
         "hkv": 4, "dh": 128, "page": 64, "causal": True},
        # the row max of one decode step, and of a packed prompt chunk
        {"name": "rowmax 1 token ctx 129", "op": "rowmax", "seqs": "1/129", "hq": 12, "causal": True},
        {"name": "rowmax prompt 16 heads", "op": "rowmax", "seqs": "1024/1024 333/1357", "hq": 16,
         "causal": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _heads(rng, most=32):
    hkv = rng.choice([1, 2, 3, 4, 8, 12])
    g = rng.choice([1, 1, 2, 3, 4, 5, 8])
    while hkv * g > most:
        g = max(1, g // 2)
        if g == 1 and hkv > most:
            hkv = most
    return hkv * g, hkv


def _seqs(rng, budget, most_q):
    """Sequence lengths with sum over sequences of q * ctx about `budget` at most."""
    n = rng.choice([1, 1, 2, 3, 5, 8])
    out = []
    for _ in range(n):
        a = 1 if rng.random() < 0.5 else _log(rng, 1, most_q)
        c = a + (0 if rng.random() < 0.4 else _log(rng, 1, 8000))
        while a * c > budget // n:
            if a > 1:
                a, c = max(1, a // 2), max(1, c // 2 + 1)
            else:
                c = max(1, c // 2)
        out.append("%d/%d" % (a, max(c, a)))
    return " ".join(out)


def draw(rng):
    op = rng.choice(["rope", "scores", "values", "rowmax"])
    hq, hkv = _heads(rng)
    dh = rng.choice([32, 40, 64, 72, 80, 96, 128])
    page = rng.choice([1, 7, 16, 32, 64, 100, 128])
    if op == "rope":
        rot = 2 * rng.randint(1, dh // 2) if rng.random() < 0.5 else dh
        tokens = _log(rng, 1, 2048)
        return {"op": op, "tokens": tokens, "hq": hq, "hkv": hkv, "dh": dh, "rot": rot,
                "interleaved": rng.random() < 0.5, "page": page, "max_pos": _log(rng, 16, 131072),
                "pad": rng.choice([0, 0, 1, 5])}
    if op == "rowmax":
        return {"op": op, "seqs": _seqs(rng, 500_000, 1024), "hq": rng.choice([1, 2, 4, 7, 12, 16]), "causal": rng.random() < 0.8}
    return {"op": op, "seqs": _seqs(rng, 240_000_000 // (hq * dh // 4), 1024), "hq": hq, "hkv": hkv, "dh": dh, "page": page,
            "causal": rng.random() < 0.8}


# ---------------------------------------------------------------------------
# shapes
# ---------------------------------------------------------------------------

def _seq_lens(case):
    """"new tokens / cached tokens, the new ones included" of every sequence."""
    pairs = [s.split("/") for s in case["seqs"].split()]
    return [int(a) for a, _ in pairs], [int(b) for _, b in pairs]


def _row_lens(case):
    """Valid keys of every row, rows in (sequence, head, query) order."""
    out = []
    for n, L in zip(*_seq_lens(case)):
        one = [max(0, min(L, L - n + i + 1)) if case["causal"] else L for i in range(n)]
        out.append(np.tile(np.asarray(one, dtype=np.int64), case["hq"]))
    return np.concatenate(out)


def _widths(lens):
    """Row widths of every round of the tournament, down to one value a row."""
    w = [lens]
    while w[-1].max(initial=0) > 1:
        w.append((w[-1] + 1) // 2)
    return w


def work(case):
    if case["op"] == "rope":
        T, hq, hkv, dh, rot = case["tokens"], case["hq"], case["hkv"], case["dh"], case["rot"]
        words = T * dh * (2 * (hq + 2 * hkv) + 2 * hq + 4 * hkv + hq + 2 * hkv)
        return {"bytes": 8 * words + T * (rot * 4 + 16), "flops": T * (hq + hkv) * rot * 2 * 3}
    lens = _row_lens(case)
    n = int(lens.sum())
    if case["op"] == "rowmax":
        w = _widths(lens)
        pairs = sum(int((a // 2).sum()) for a in w[:-1])
        # the scores once for the rounds and once for the difference, the gates' shares in,
        # the opened differences and both parties' results out
        return {"bytes": 8 * (2 * n + 2 * n + 2 * n + 2 * pairs + pairs), "flops": 2 * n + 4 * pairs}
    (q, ctx), hq, hkv, dh = _seq_lens(case), case["hq"], case["hkv"], case["dh"]
    T, cache = sum(q), 3 * sum(ctx) * hkv * dh
    per_row = 3 if case["op"] == "scores" else 4
    return {"bytes": 8 * (cache + 3 * T * hq * dh + per_row * n + (T * hq * dh if case["op"] == "values" else 0)),
            "flops": 2 * 2 * n * dh}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _u64(g, *shape):
    """Uniform 64-bit words (masks and shares), as int64."""
    return torch.randint(-(2**63), 2**63 - 1, shape, dtype=torch.int64, device=g.device, generator=g)


def _fixed(g, sigma, *shape):
    """Gaussian values in fixed point."""
    return (torch.randn(shape, generator=g, device=g.device) * (sigma * 2**F)).round().to(torch.int64)


def _shared(g, x):
    s = _u64(g, *x.shape)
    return s, x - s


def _limbs(x):
    """16-bit limbs of 64-bit words, as float64 matrices."""
    return [((x >> (16 * i)) & 0xFFFF).to(torch.float64) for i in range(4)]


def _mm(a, b):
    """a @ b mod 2^64 for int64 matrices: ten products of 16-bit limbs, each
    exact in float64 up to a depth of 2^19."""
    la, lb = _limbs(a), _limbs(b)
    out = None
    for s in range(4):
        p = la[0] @ lb[s]
        for i in range(1, s + 1):
            p = p + la[i] @ lb[s - i]
        p = p.to(torch.int64) << (16 * s)
        out = p if out is None else out + p
    return out


def _pages(case, g):
    """A pool a little larger than the sequences need, its pages dealt out in
    random order: (pool pages, block table [sequences][most pages])."""
    page = case["page"]
    need = [-(-L // page) for L in _seq_lens(case)[1]]
    total = sum(need)
    pool = total + 2
    order = torch.randperm(pool, device=g.device, generator=g).to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device=g.device)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return pool, table


def _sequence(st, pool, b):
    """Sequence b's cached words [heads][tokens][head size] out of the pages."""
    L, page = _seq_lens(st["case"])[1][b], st["case"]["page"]
    ids = st["table"][b, :-(-L // page)].long()
    return pool[ids].transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :L]


def _rows(st):
    """(sequence, first token, queries, context, first packed word of the sequence)."""
    at = t = 0
    c = st["case"]
    for b, (n, L) in enumerate(zip(*_seq_lens(c))):
        yield b, t, n, L, at
        if c["causal"]:
            at += c["hq"] * sum(max(0, L - n + i + 1) for i in range(n))
        else:
            at += c["hq"] * n * L
        t += n


def _mask(n, L, causal, dev):
    """[queries][keys]: which keys a query sees."""
    if not causal:
        return torch.ones((n, L), dtype=torch.bool, device=dev)
    return torch.arange(L, device=dev)[None, :] <= (L - n + torch.arange(n, device=dev))[:, None]


def _by_kv(x, hkv):
    """[queries][heads][size] -> [key heads][heads of the group x queries][size]."""
    n, hq, size = x.shape
    return x.transpose(0, 1).reshape(hkv, hq // hkv * n, size)


def _dense(packed, at, m, hq):
    """The packed rows of one sequence as [heads][queries][keys], zero where masked."""
    each = int(m.sum())
    full = torch.zeros((hq,) + tuple(m.shape), dtype=torch.int64, device=m.device)
    full[:, m] = packed[at:at + hq * each].view(hq, each)
    return full


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = _gen(seed, dev)
    st = {"case": case}
    if case["op"] == "rope":
        _prepare_rope(case, st, g, seed)
    elif case["op"] == "rowmax":
        _prepare_rowmax(case, st, g, seed)
    else:
        _prepare_attention(case, st, g, seed)
    return st


def _prepare_rope(case, st, g, seed):
    dev = g.device
    T, hq, hkv, dh, page = case["tokens"], case["hq"], case["hkv"], case["dh"], case["page"]
    # both parties' fused rows of queries, keys and values, as a projection leaves them
    qkv = _shared(g, _fixed(g, 1.0, T, (hq + 2 * hkv) * dh))
    st["qkv"] = qkv
    st["q"] = tuple(x[:, :hq * dh].view(T, hq, dh) for x in qkv)
    st["k"] = tuple(x[:, hq * dh:(hq + hkv) * dh].view(T, hkv, dh) for x in qkv)
    st["v"] = tuple(x[:, (hq + hkv) * dh:].view(T, hkv, dh) for x in qkv)
    st["a"] = (_u64(g, T, hq, dh), _u64(g, T, hq, dh))
    pool = -(-T // page) + 2
    for name in ("ek", "ev", "bk0", "bk1", "bv0", "bv1"):
        st[name] = _u64(g, pool, hkv, page, dh)
    st["slots"] = torch.randperm(pool * page, device=dev, generator=g)[:T].to(torch.int64)
    pos = torch.randint(0, case["max_pos"], (T,), device=dev, generator=g, dtype=torch.int64).to(torch.int32)
    pad = min(case["pad"], T - 1)
    if pad:
        st["slots"][T - pad:] = -1  # padding rows behind the last sequence
    st["pos"] = pos
    # cosines and sines in fixed point, the frequencies of a long-context model (base 500,000)
    half = case["rot"] // 2
    inv = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
    ang = torch.arange(case["max_pos"], dtype=torch.float64, device=dev)[:, None] * inv[None, :]
    st["cos"] = (ang.cos() * 2**F).round().to(torch.int32)
    st["sin"] = (ang.sin() * 2**F).round().to(torch.int32)
    st["dq"] = torch.zeros((T, hq, dh), dtype=torch.int64, device=dev)
    if own:
        from suf_b200.attention import ShareCache, TruncPair

        st["trunc"] = TruncPair(_ctx(), F, seed=seed & 0xFFFFFFFF)
        st["cache"] = ShareCache.from_tensors(_ctx(), st["ek"], (st["bk0"], st["bk1"]), st["ev"],
                                              (st["bv0"], st["bv1"]))


def _prepare_attention(case, st, g, seed):
    dev = g.device
    T, hq, hkv, dh, page = sum(_seq_lens(case)[0]), case["hq"], case["hkv"], case["dh"], case["page"]
    pool, st["table"] = _pages(case, g)
    b0, b1 = _u64(g, pool, hkv, page, dh), _u64(g, pool, hkv, page, dh)
    # the cached entries are X - B for keys or values X of unit size
    st["e"] = _fixed(g, 1.0, pool, hkv, page, dh) - b0 - b1
    st["b"] = (b0, b1)
    st["r"] = (seed * 0x9E3779B97F4A7C15 % 2**64, seed * 0xD1B54A32D192ED03 % 2**64)
    if case["op"] == "scores":
        a = _u64(g, T, hq, dh)
        st["a"] = _shared(g, a)
        st["dq"] = _fixed(g, 1.0, T, hq, dh) - a
        parts = []
        for b, t, n, L, _ in _rows(st):
            m = _mask(n, L, case["causal"], dev)
            bb = _sequence(st, b0, b) + _sequence(st, b1, b)
            z = _mm(_by_kv(a[t:t + n], hkv), bb.transpose(1, 2))
            parts.append(z.view(hq, n, L)[:, m].flatten())
        st["c"] = _shared(g, torch.cat(parts))
        st["out"] = torch.empty_like(st["c"][0])
    else:
        n_words = int(_row_lens(case).sum())
        # probabilities: non-negative, of the size of an even spread over the row
        p = (torch.rand(n_words, device=dev, generator=g) * 2 ** (F - 2)).to(torch.int64)
        st["p"] = _shared(g, p)
        a = _u64(g, n_words)
        st["a"] = _shared(g, a)
        c = torch.empty((T, hq, dh), dtype=torch.int64, device=dev)
        for b, t, n, L, at in _rows(st):
            m = _mask(n, L, case["causal"], dev)
            bb = _sequence(st, b0, b) + _sequence(st, b1, b)
            z = _mm(_dense(a, at, m, hq).view(hkv, -1, L), bb)
            c[t:t + n] = z.view(hq, n, dh).transpose(0, 1)
        st["c"] = _shared(g, c)
        st["out"] = torch.empty_like(st["c"][0])
    if own:
        from suf_b200.attention import AttnLayout

        st["layout"] = AttnLayout(_ctx(), *_seq_lens(case), st["table"], page, hq, hkv, causal=case["causal"])


def _prepare_rowmax(case, st, g, seed):
    lens = _row_lens(case)
    n = int(lens.sum())
    st["lens"] = lens
    st["widths"] = _widths(lens)
    st["s"] = _shared(g, _fixed(g, 2.0, n))
    # what the ReLU gates between the rounds answer with: shares, one per pair
    st["relu"] = [_shared(g, _fixed(g, 1.0, int((w // 2).sum())).abs()) for w in st["widths"][:-1]]
    st["r"] = [((seed + 2 * i + 1) * 0x9E3779B97F4A7C15 % 2**64, (seed + i) * 0xD1B54A32D192ED03 % 2**64)
               for i in range(len(st["relu"]))]
    # row of every packed value, per round
    st["row"] = [torch.from_numpy(np.repeat(np.arange(lens.size), w)).to(g.device) for w in st["widths"]]
    st["off"] = [torch.from_numpy(np.concatenate([[0], np.cumsum(w)])).to(g.device) for w in st["widths"]]
    if own:
        from suf_b200.attention import RowMaxPlan

        st["plan"] = RowMaxPlan(_ctx(), lens)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _signed(x):
    """A word as the int64 of the same bits."""
    x %= 2**64
    return x - 2**64 if x >= 2**63 else x


def _plain_rope(st):
    c = st["case"]
    half, page = c["rot"] // 2, c["page"]
    keep = st["slots"] >= 0
    cos = st["cos"][st["pos"].long()].long()[:, None, :]
    sin = st["sin"][st["pos"].long()].long()[:, None, :]

    def rotate(x):
        y = x.clone()
        if c["interleaved"]:
            x1, x2 = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
            y[..., 0:2 * half:2] = (x1 * cos - x2 * sin) >> F
            y[..., 1:2 * half:2] = (x2 * cos + x1 * sin) >> F
        else:
            x1, x2 = x[..., :half], x[..., half:2 * half]
            y[..., :half] = (x1 * cos - x2 * sin) >> F
            y[..., half:2 * half] = (x2 * cos + x1 * sin) >> F
        return y

    st["dq"][keep] = (rotate(st["q"][0] + st["q"][1]) - st["a"][0] - st["a"][1])[keep]
    at, slot = torch.div(st["slots"][keep], page, rounding_mode="floor"), st["slots"][keep] % page
    k, v = rotate(st["k"][0] + st["k"][1])[keep], (st["v"][0] + st["v"][1])[keep]
    st["ek"][at, :, slot] = k - st["bk0"][at, :, slot] - st["bk1"][at, :, slot]
    st["ev"][at, :, slot] = v - st["bv0"][at, :, slot] - st["bv1"][at, :, slot]
    return st["dq"], st["ek"], st["ev"]


def _own_rope(st):
    from suf_b200.attention import rope_append_pair

    rope_append_pair(_ctx(), st["q"], st["k"], st["v"], st["pos"], st["slots"], st["cos"], st["sin"], st["trunc"],
                     st["a"], st["cache"], st["dq"], interleaved=st["case"]["interleaved"])
    return st["dq"], st["ek"], st["ev"]


def _plain_scores(st):
    c = st["case"]
    parts = []
    for b, t, n, L, _ in _rows(st):
        m = _mask(n, L, c["causal"], st["e"].device)
        e = _sequence(st, st["e"], b)
        bb = _sequence(st, st["b"][0], b) + _sequence(st, st["b"][1], b)
        d, u = st["dq"][t:t + n], (st["dq"] + st["a"][0] + st["a"][1])[t:t + n]
        # D B + (A + D) E, one product of twice the depth
        z = _mm(_by_kv(torch.cat([d, u], dim=2), c["hkv"]), torch.cat([bb, e], dim=2).transpose(1, 2))
        parts.append(z.view(c["hq"], n, L)[:, m].flatten())
    return torch.cat(parts) + st["c"][0] + st["c"][1] + _signed(st["r"][0] + st["r"][1])


def _own_scores(st):
    from suf_b200.attention import attn_scores_pair

    return attn_scores_pair(_ctx(), st["dq"], st["a"], st["c"], st["r"], st["e"], st["b"], st["layout"],
                            out=st["out"])


def _plain_values(st):
    c = st["case"]
    d = st["p"][0] + st["p"][1] - st["a"][0] - st["a"][1]
    u = d + st["a"][0] + st["a"][1]
    out = st["c"][0] + st["c"][1] + _signed(st["r"][0] + st["r"][1])
    for b, t, n, L, at in _rows(st):
        m = _mask(n, L, c["causal"], st["e"].device)
        e = _sequence(st, st["e"], b)
        bb = _sequence(st, st["b"][0], b) + _sequence(st, st["b"][1], b)
        left = torch.cat([_dense(x, at, m, c["hq"]).view(c["hkv"], -1, L) for x in (d, u)], dim=2)
        z = _mm(left, torch.cat([bb, e], dim=1))
        out[t:t + n] += z.view(c["hq"], n, c["dh"]).transpose(0, 1)
    return out


def _own_values(st):
    from suf_b200.attention import attn_values_pair

    return attn_values_pair(_ctx(), st["p"], st["a"], st["c"], st["r"], st["e"], st["b"], st["layout"],
                            out=st["out"])


def _plain_rowmax(st):
    cur = st["s"]
    opened = []
    for k, (relu, r) in enumerate(zip(st["relu"], st["r"])):
        w = st["off"][k][1:] - st["off"][k][:-1]
        prow = torch.repeat_interleave(torch.arange(w.numel(), device=w.device), w // 2)
        first = torch.cumsum(w // 2, 0) - w // 2
        at = st["off"][k][prow] + 2 * (torch.arange(prow.numel(), device=w.device) - first[prow])
        opened.append((cur[0][at] - cur[0][at + 1]) + (cur[1][at] - cur[1][at + 1]) + _signed(r[0] + r[1]))
        # the winners, and the value left over at the end of an odd row
        j = torch.arange(st["row"][k + 1].numel(), device=w.device) - st["off"][k + 1][st["row"][k + 1]]
        row = st["row"][k + 1]
        src = st["off"][k][row] + 2 * j
        last = 2 * j + 1 >= w[row]
        pair = (first[row] + j).clamp(max=max(prow.numel() - 1, 0))
        cur = tuple(torch.where(last, c[src], c[torch.where(last, src, src + 1)] + q[pair])
                    for c, q in zip(cur, relu))
    has = torch.cumsum((st["off"][0][1:] > st["off"][0][:-1]).long(), 0) - 1
    return opened, [m[has[st["row"][0]]] - s for m, s in zip(cur, st["s"])]


def _own_rowmax(st):
    from suf_b200.attention import maxdiff_ragged_pair, rowmax_open_pair, rowmax_round_pair

    plan, opened, cur = st["plan"], [], st["s"]
    if st["relu"]:
        opened.append(rowmax_open_pair(_ctx(), plan, cur, st["r"][0]))
    for k, relu in enumerate(st["relu"]):
        nxt = st["r"][k + 1] if k + 1 < len(st["r"]) else None
        cur, xhat = rowmax_round_pair(_ctx(), plan, k, cur, relu, nxt)
        if xhat is not None:
            opened.append(xhat)
    return opened, list(maxdiff_ragged_pair(_ctx(), plan, cur, st["s"]))


_plain = {"rope": _plain_rope, "scores": _plain_scores, "values": _plain_values, "rowmax": _plain_rowmax}
_own = {"rope": _own_rope, "scores": _own_scores, "values": _own_values, "rowmax": _own_rowmax}


# ---------------------------------------------------------------------------
# the definition, word by word on the host
# ---------------------------------------------------------------------------

def _np(t):
    return t.cpu().numpy().view(np.uint64) if t.dtype == torch.int64 else t.cpu().numpy()


def exact(case, seed):
    """The definition in numpy's 64-bit words; None where its integer products
    (about half a billion a second) would take too long."""
    if case["op"] == "rope":
        return _exact_rope(prepare(case, seed))
    if case["op"] == "rowmax":
        return _exact_rowmax(prepare(case, seed))
    pairs = sum(n * L for n, L in zip(*_seq_lens(case))) * case["hq"] * case["dh"]
    if pairs > 3e9:
        return None
    return _exact_attention(prepare(case, seed))


def _exact_rope(st):
    c = st["case"]
    half, page, dh = c["rot"] // 2, c["page"], c["dh"]
    slots, pos = st["slots"].cpu().numpy(), st["pos"].cpu().numpy()
    cos, sin = st["cos"].cpu().numpy().astype(np.int64), st["sin"].cpu().numpy().astype(np.int64)
    dq, ek, ev = (_np(st[k]).copy() for k in ("dq", "ek", "ev"))
    first = np.arange(half) * 2 if c["interleaved"] else np.arange(half)
    second = first + 1 if c["interleaved"] else first + half
    masks = [_np(st[k]) for k in ("bk0", "bk1", "bv0", "bv1")]
    qkv = [_np(x) for x in st["qkv"]]
    a = [_np(x) for x in st["a"]]
    with np.errstate(over="ignore"):
        for t in range(c["tokens"]):
            if slots[t] < 0:
                continue
            # add the shares as words, read the sum as signed
            x = (qkv[0][t] + qkv[1][t]).view(np.int64).reshape(-1, dh)
            turn = x[:c["hq"] + c["hkv"]].copy()
            x1, x2 = turn[:, first].copy(), turn[:, second].copy()
            co, si = cos[pos[t]], sin[pos[t]]
            turn[:, first] = np.floor_divide(x1 * co - x2 * si, 2**F)
            turn[:, second] = np.floor_divide(x2 * co + x1 * si, 2**F)
            page_at, at = divmod(int(slots[t]), page)
            dq[t] = turn[:c["hq"]].view(np.uint64) - a[0][t] - a[1][t]
            ek[page_at, :, at] = turn[c["hq"]:].view(np.uint64) - masks[0][page_at, :, at] - masks[1][page_at, :, at]
            ev[page_at, :, at] = (x[c["hq"] + c["hkv"]:].view(np.uint64) - masks[2][page_at, :, at] -
                                  masks[3][page_at, :, at])
    return dq.view(np.int64), ek.view(np.int64), ev.view(np.int64)


def _exact_attention(st):
    c = st["case"]
    scores = c["op"] == "scores"
    page, group, dh = c["page"], c["hq"] // c["hkv"], c["dh"]
    table = st["table"].cpu().numpy()
    e, b0, b1 = _np(st["e"]), _np(st["b"][0]), _np(st["b"][1])
    c0, c1 = _np(st["c"][0]), _np(st["c"][1])
    a0, a1 = _np(st["a"][0]), _np(st["a"][1])
    r = [np.uint64(v) for v in st["r"]]
    dq = _np(st["dq"]) if scores else None
    p0, p1 = (None, None) if scores else (_np(x) for x in st["p"])
    out = np.empty_like(c0)
    at = t = 0
    with np.errstate(over="ignore"):
        for b, (n, L) in enumerate(zip(*_seq_lens(c))):
            where = [(int(table[b, j // page]), j % page) for j in range(L)]
            ids, offs = np.array([w[0] for w in where], dtype=np.int64), np.array([w[1] for w in where], dtype=np.int64)
            for h in range(c["hq"]):
                ee, m0, m1 = (x[ids, h // group, offs] for x in (e, b0, b1))
                for i in range(n):
                    m = max(0, L - n + i + 1) if c["causal"] else L
                    if scores:
                        d, u0, u1 = dq[t + i, h], a0[t + i, h], a1[t + i, h]
                        z0 = c0[at:at + m] + m0[:m] @ d + ee[:m] @ u0 + ee[:m] @ d
                        z1 = c1[at:at + m] + m1[:m] @ d + ee[:m] @ u1
                        out[at:at + m] = (z0 + r[0]) + (z1 + r[1])
                    else:
                        w = slice(at, at + m)
                        d = (p0[w] - a0[w]) + (p1[w] - a1[w])
                        z0 = c0[t + i, h] + d @ m0[:m] + a0[w] @ ee[:m] + d @ ee[:m]
                        z1 = c1[t + i, h] + d @ m1[:m] + a1[w] @ ee[:m]
                        out[t + i, h] = (z0 + r[0]) + (z1 + r[1])
                    at += m
            t += n
    return out.view(np.int64)


def _exact_rowmax(st):
    cur = [_np(x) for x in st["s"]]
    lens = st["lens"]
    if lens.size > 60000:
        return None
    opened = []
    rows = [np.split(x, np.cumsum(lens)[:-1]) for x in cur]
    base = [list(x) for x in rows]
    with np.errstate(over="ignore"):
        for relu, r in zip(st["relu"], st["r"]):
            add = np.uint64(r[0]), np.uint64(r[1])
            got = [_np(x) for x in relu]
            at, diffs, nxt = 0, [], [[], []]
            for a, b in zip(*rows):
                k = a.size // 2
                diffs.append((a[0:2 * k:2] - a[1:2 * k:2] + add[0]) + (b[0:2 * k:2] - b[1:2 * k:2] + add[1]))
                for p, x in ((0, a), (1, b)):
                    nxt[p].append(np.concatenate([x[1:2 * k:2] + got[p][at:at + k], x[2 * k:]]))
                at += k
            opened.append(np.concatenate(diffs).view(np.int64))
            rows = nxt
        t = [np.concatenate([m[0] - s if s.size else s for m, s in zip(rows[p], base[p])]) for p in (0, 1)]
    return opened, [x.view(np.int64) for x in t]
