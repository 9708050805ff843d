"""CPU tests of attention over a cache of shares: the kernels' address
arithmetic (a CPU build of the same code), the refusals of the C entries
(a host-only context: a call with good arguments gets as far as "no device")
and of the Python wrappers, and the rotary tables."""
from __future__ import annotations

import ctypes as C
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def emu(tmp_path_factory):
    out = tmp_path_factory.mktemp("attn_emu") / "libattn.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-I/usr/local/cuda/include", "-o", str(out),
                    str(ROOT / "tests" / "hostemu" / "attn_shim.cpp")], check=True)
    E = C.CDLL(str(out))
    E.emu_row_off.restype = C.c_int64
    E.emu_page_word.restype = C.c_int64
    E.emu_sizeof.restype = C.c_size_t
    E.emu_seq_fits.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int64, C.c_void_p]
    E.emu_page_word.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int]
    return E


def test_struct_mirrors(emu):
    from suf_b200._lib import AttnSeqs, RopeAppend

    assert emu.emu_sizeof(0) == C.sizeof(RopeAppend) and emu.emu_sizeof(1) == C.sizeof(AttnSeqs)


@pytest.mark.parametrize("causal", [0, 1])
def test_row_offsets_match_brute_force(emu, causal):
    for n in range(0, 9):
        for L in range(0, 12):
            lens = [max(0, L - n + i + 1) if causal else L for i in range(n)]
            assert [emu.emu_row_len(n, L, causal, i) for i in range(n)] == lens
            assert [emu.emu_row_off(n, L, causal, i) for i in range(n + 1)] == [sum(lens[:i]) for i in range(n + 1)]
    # past 32 bits
    n, L = 100_000, 200_000
    want = sum(L - n + i + 1 for i in range(n)) if causal else n * L
    assert want > 2**33 and emu.emu_row_off(n, L, causal, n) == want


def _seqs(**kw):
    from suf_b200._lib import AttnSeqs

    s = AttnSeqs()
    for k, v in dict(tokens=10, cached=60, packed=1000, batch=2, max_pages=4, page_size=8, pages=5, q_heads=4, kv_heads=2,
                     head_dim=64, causal=1, min_q=1, max_q=6, max_ctx=30).items():
        setattr(s, k, v)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_sequences_outside_the_host_bounds_are_refused(emu):
    s, blk = _seqs(), C.c_int64()

    def fits(*a):
        return emu.emu_seq_fits(C.byref(s), *a, C.byref(blk))

    assert fits(0, 6, 0, 30, 0) and blk.value == sum(range(25, 31))
    assert fits(4, 10, 54, 60, 1000 - 4 * 21)
    for bad in [(-1, 3, 0, 5, 0), (3, 2, 0, 5, 0), (5, 11, 0, 5, 0), (0, 7, 0, 5, 0), (0, 3, 5, 4, 0), (0, 3, 0, 31, 0),
                (0, 3, 0, 5, -1), (0, 3, 0, 5, 1001), (4, 10, 0, 6, 1000 - 4 * 21 + 1), (0, 3, 56, 61, 0),
                (0, 3, -1, 4, 0), (-2**31, 2**31 - 1, -2**31, 2**31 - 1, 0), (0, 2**31 - 1, 0, 2**31 - 1, 2**63 - 1)]:
        assert not fits(*bad), bad
    s.max_ctx = 40
    assert not fits(0, 3, 0, 33, 0)  # more than four pages of eight


def test_pages_outside_the_pool_are_refused(emu):
    s = _seqs()
    assert emu.emu_page_word(C.byref(s), 0, 0, 0) == 0
    assert emu.emu_page_word(C.byref(s), 4, 1, 13) == ((4 * 2 + 1) * 8 + 5) * 64
    for pg in (-1, 5, 2**31 - 1, -2**31):
        assert emu.emu_page_word(C.byref(s), pg, 0, 0) == -1
    # a long cache: offsets past 32 bits
    s.pages, s.kv_heads, s.page_size, s.head_dim = 10**6, 8, 64, 128
    assert emu.emu_page_word(C.byref(s), 10**6 - 1, 7, 63) == 10**6 * 8 * 64 * 128 - 128


def test_blocks_of_packed_sequences_never_overlap(emu):
    """Every sequence has room for all its blocks before the next one starts,
    and the last one within the bound that sizes grids and workspaces."""
    emu.emu_first_block.restype = emu.emu_blocks_of.restype = C.c_int64
    emu.emu_first_block.argtypes, emu.emu_blocks_of.argtypes = [C.c_int64, C.c_int, C.c_int], [C.c_int64, C.c_int, C.c_int]
    rng = np.random.default_rng(1)
    for _ in range(300):
        per, m = int(rng.choice([32, 64, 128])), int(rng.choice([1, 4, 5]))
        lens = rng.choice([0, 1, 7, 31, 32, 33, 64, 127, 128, 129, 500], rng.integers(1, 9)) * m
        at = np.concatenate([[0], np.cumsum(lens)])
        end = 0
        for b, n in enumerate(lens):
            first = emu.emu_first_block(int(at[b]), b, per)
            assert first >= end
            end = first + -(-int(n) // per)
        assert end <= emu.emu_blocks_of(int(at[-1]), len(lens), per)


# -- refusals of the C entries ----------------------------------------------------

@pytest.fixture(scope="module")
def host():
    from suf_b200 import _lib
    from suf_b200.build import build

    build()
    h = C.c_void_p()
    _lib.check(_lib.lib().sufb200_ctx_create(-1, C.byref(h)))
    yield h
    _lib.lib().sufb200_ctx_destroy(h)


P16, P8, P4 = 0x10000, 0x10008, 0x10004  # addresses the refused calls never touch


def _arr(*v):
    return (C.c_void_p * 2)(*v)


def _attn(host, which, seqs, x=None, a=(P16, P16), c=(P16, P16), e=P16, b=(P16, P16), out=P16, r=(1, 2)):
    from suf_b200 import _lib

    L = _lib.lib()
    rr = (C.c_uint64 * 2)(*r)
    if which == "scores":
        return L.sufb200_attn_scores_pair(host, C.byref(seqs), P16 if x is None else x, _arr(*a), _arr(*c), rr, e,
                                          _arr(*b), out, None)
    return L.sufb200_attn_values_pair(host, C.byref(seqs), _arr(*(x or (P16, P16))), _arr(*a), _arr(*c), rr, e,
                                      _arr(*b), out, None)


PTRS = dict(d_cu_q=P16, d_cu_ctx=P16, d_row_base=P16, d_block_table=P16)


@pytest.mark.parametrize("which", ["scores", "values"])
def test_attention_refusals(host, which):
    from suf_b200 import _lib

    ok = _seqs(**PTRS)
    assert _attn(host, which, ok) == _lib.ERR_UNSUPPORTED  # good arguments: only the device is missing
    assert b"host-only" in _lib.lib().sufb200_last_error()
    for bad, code in [(dict(head_dim=63), _lib.ERR_UNSUPPORTED), (dict(head_dim=258), _lib.ERR_UNSUPPORTED),
                      (dict(head_dim=0), _lib.ERR_UNSUPPORTED), (dict(q_heads=3), _lib.ERR_INVALID),
                      (dict(kv_heads=0), _lib.ERR_INVALID), (dict(page_size=0), _lib.ERR_INVALID),
                      (dict(max_ctx=33), _lib.ERR_INVALID), (dict(batch=-1), _lib.ERR_INVALID),
                      (dict(tokens=-1), _lib.ERR_INVALID), (dict(n_tiles=3), _lib.ERR_INVALID),
                      (dict(min_q=7), _lib.ERR_INVALID), (dict(cached=-1), _lib.ERR_INVALID), (dict(d_cu_ctx=None), _lib.ERR_INVALID),
                      (dict(d_block_table=None), _lib.ERR_INVALID), (dict(batch=40000), _lib.ERR_UNSUPPORTED),
                      (dict(max_q=2**20), _lib.ERR_UNSUPPORTED), (dict(tokens=2**31), _lib.ERR_UNSUPPORTED),
                      (dict(cached=2**31), _lib.ERR_UNSUPPORTED),
                      (dict(max_ctx=2**26 + 1, max_pages=2**26), _lib.ERR_UNSUPPORTED),
                      (dict(q_heads=2**20, kv_heads=2**16 - 1 + 1, batch=1), _lib.ERR_UNSUPPORTED)]:
        assert _attn(host, which, _seqs(**{**PTRS, **bad})) == code, bad
        assert b"head" in _lib.lib().sufb200_last_error() or b"attn_" in _lib.lib().sufb200_last_error()
    for kw in [dict(a=(P16, None)), dict(c=(P4, P16)), dict(out=None), dict(out=P4), dict(e=P8), dict(b=(P16, P8)),
               dict(e=None)]:
        assert _attn(host, which, ok, **kw) == _lib.ERR_INVALID, kw
    assert _attn(host, which, _seqs(**{**PTRS, "batch": 0})) == _lib.OK  # nothing to do


def _rope(**kw):
    from suf_b200._lib import RopeAppend

    a = RopeAppend()
    for f in ("d_q", "d_k", "d_v", "d_a", "d_bk", "d_bv", "d_tables"):
        setattr(a, f, _arr(P16, P16))
    for f in ("d_positions", "d_slots", "d_cos", "d_sin", "d_dq", "d_ek", "d_ev"):
        setattr(a, f, P16)
    for k, v in dict(tokens=3, q_heads=4, kv_heads=2, head_dim=64, rot_dim=64, max_pos=16, pages=2,
                     page_size=8).items():
        setattr(a, k, v)
    for p in (0, 1):
        d = a.trunc[p]
        d.kind, d.frac_bits, d.party, d.nq, d.carry_a, d.carry_b = 2, 12, p, 2, 0, 1
        d.q_bits[0] = d.q_bits[1] = 12
        d.sign_a = d.sign_b = d.wrap_q = -1
    for k, v in kw.items():
        if k in ("kind", "frac_bits", "party", "carry_a", "nq"):
            setattr(a.trunc[1], k, v)
        else:
            setattr(a, k, v)
    return a


def test_rope_append_refusals(host):
    from suf_b200 import _lib

    L = _lib.lib()

    def call(**kw):
        a = _rope(**kw)
        return L.sufb200_rope_append_pair(host, C.byref(a), None)

    assert call() == _lib.ERR_UNSUPPORTED and b"host-only" in L.sufb200_last_error()
    assert call(tokens=0) == _lib.OK
    assert call(carry_a=-1, nq=0, d_tables=_arr(P16, None)) == _lib.ERR_UNSUPPORTED  # no queries: no tables
    assert call(q_heads=0, d_q=_arr(None, None), d_a=_arr(None, None), d_dq=None) == _lib.ERR_UNSUPPORTED
    assert call(rot_dim=0, d_positions=None, d_cos=None, d_sin=None, d_tables=_arr(None, None)) == _lib.ERR_UNSUPPORTED
    for kw in [dict(tokens=-1), dict(kv_heads=0), dict(page_size=0), dict(pages=0), dict(rot_dim=66), dict(rot_dim=3),
               dict(d_slots=None), dict(d_k=_arr(P16, None)), dict(d_q=_arr(P16, None)), dict(d_a=_arr(P4, P16)),
               dict(d_bv=_arr(P4, P16)), dict(d_dq=None), dict(d_ek=P4), dict(d_positions=None), dict(d_cos=None),
               dict(max_pos=0), dict(kind=1), dict(frac_bits=11), dict(party=0), dict(carry_a=2), dict(nq=5),
               dict(d_tables=_arr(P16, None)), dict(d_tables=_arr(P16, P8))]:
        assert call(**kw) == _lib.ERR_INVALID, kw
    assert call(head_dim=65) == _lib.ERR_UNSUPPORTED
    assert L.sufb200_rope_append_pair(host, None, None) == _lib.ERR_INVALID


def test_rowmax_refusals(host):
    from suf_b200 import _lib

    L = _lib.lib()
    r = (C.c_uint64 * 2)(1, 2)
    g = _arr(P16, P16)
    assert L.sufb200_rowmax_open_pair(host, g, 4, 9, P16, P16, r, P16, None) == _lib.ERR_UNSUPPORTED
    assert L.sufb200_rowmax_open_pair(host, g, 0, 9, P16, P16, r, P16, None) == _lib.OK
    assert L.sufb200_rowmax_open_pair(host, g, 4, 1, P16, P16, r, P16, None) == _lib.OK
    for args in [(None, 4, 9, P16, P16, r, P16), (g, -1, 9, P16, P16, r, P16), (g, 4, 9, None, P16, r, P16),
                 (g, 4, 9, P16, P16, None, P16), (g, 4, 9, P16, P16, r, P4), (_arr(P16, None), 4, 9, P16, P16, r, P16)]:
        assert L.sufb200_rowmax_open_pair(host, *args, None) == _lib.ERR_INVALID, args
    assert L.sufb200_rowmax_round_pair(host, g, g, 4, 9, P16, P16, P16, r, g, P16, None) == _lib.ERR_UNSUPPORTED
    assert L.sufb200_rowmax_round_pair(host, g, g, 4, 9, P16, P16, None, None, g, None, None) == _lib.ERR_UNSUPPORTED
    for args in [(g, _arr(None, P16), 4, 9, P16, P16, P16, r, g, P16), (g, g, 4, 9, P16, P16, None, r, g, P16),
                 (g, g, 4, 9, P16, P16, P16, None, g, P16), (g, g, 4, 9, P16, P16, P16, r, _arr(P16, P4), P16),
                 (g, g, 4, -1, P16, P16, P16, r, g, P16)]:
        assert L.sufb200_rowmax_round_pair(host, *args, None) == _lib.ERR_INVALID, args
    assert L.sufb200_maxdiff_ragged_pair(host, g, g, 4, 9, P16, P16, g, None) == _lib.ERR_UNSUPPORTED
    for args in [(g, g, 4, 9, P16, None, g), (g, _arr(None, P16), 4, 9, P16, P16, g), (g, g, -4, 9, P16, P16, g)]:
        assert L.sufb200_maxdiff_ragged_pair(host, *args, None) == _lib.ERR_INVALID, args


# -- refusals of the wrappers ---------------------------------------------------------

class _Ctx:
    device = 0


def test_wrappers_refuse_wrong_tensors():
    import torch

    from suf_b200 import attention as at

    x = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="cuda:0"):
        at._want(_Ctx, "x", x, (4,))
    with pytest.raises(ValueError, match="int64"):
        at._want(_Ctx, "x", x.to(torch.int32), (4,))
    with pytest.raises(ValueError, match="both parties"):
        at._pair(_Ctx, "x", x, (4,))
    with pytest.raises(ValueError, match="both parties"):
        at._masks((1,))
    with pytest.raises(ValueError, match="cuda:0"):
        at._strided(_Ctx, "q", (torch.zeros(1, 2, 4, dtype=torch.int64),) * 2, (1, 2, 4))
    for bad in [dict(rot_dim=3), dict(max_pos=0), dict(frac_bits=0), dict(frac_bits=17), dict(scale=0.0),
                dict(base=-1.0), dict(low_freq=1.0), dict(low_freq=2.0, high_freq=1.0, trained_pos=64)]:
        with pytest.raises(ValueError):
            at.rope_table_words(**{**dict(max_pos=8, rot_dim=4, frac_bits=12), **bad})


def test_rope_tables_are_rounded_cosines_of_the_definition():
    """Every entry is the nearest fixed-point value of the exact cosine or sine:
    off by at most half a unit, plus the float64 angle's own error (position
    131071 times a frequency: 2^17 * 2^-53 in the angle, 2^-24 units at 12 bits)."""
    from suf_b200.attention import rope_table_words

    cos, sin = rope_table_words(131072, 8, 12, base=500000.0, scale=4.0)
    for pos in (0, 1, 77, 4095, 131071):
        for i in range(4):
            ang = math.fmod(pos * 500000.0 ** (-i / 4) / 4.0, 2 * math.pi)
            assert abs(cos[pos, i] - 4096 * math.cos(ang)) <= 0.5 + 2**-20
            assert abs(sin[pos, i] - 4096 * math.sin(ang)) <= 0.5 + 2**-20
    # blended scaling: fast pairs stay, slow pairs are stretched, between them a blend
    plain, _ = rope_table_words(512, 16, 12)
    all_, _ = rope_table_words(512, 16, 12, scale=8.0)
    mix, _ = rope_table_words(512, 16, 12, scale=8.0, low_freq=1.0, high_freq=4.0, trained_pos=256)
    turns = 256 * 10000.0 ** (-np.arange(8) / 8) / (2 * math.pi)
    assert (turns > 4).any() and (turns < 1).any() and ((turns > 1) & (turns < 4)).any()
    for i in range(8):
        if turns[i] >= 4:
            assert (mix[:, i] == plain[:, i]).all()
        elif turns[i] <= 1:
            assert (mix[:, i] == all_[:, i]).all()
        else:
            assert (mix[:, i] != plain[:, i]).any() and (mix[:, i] != all_[:, i]).any()


def test_mma_order_covers_every_limb_pair_once():
    """The tensor-core kernels' twelve MMAs of a step (attention_tc.cu): every
    limb pair (i, j), i + j <= 7, once on its diagonal, within the 512 columns,
    the two that start from zero first and covering all of them."""
    import re

    src = (ROOT / "suf_b200" / "csrc" / "attention_tc.cu").read_text()
    calls = [(int(i), int(j), acc) for i, j, acc in re.findall(r"issue_one\(al, bl, (\d), (\d), (accumulate|1u)\);", src)]
    assert "const int n = 64 * (8 - i - j);" in src and "idesc_n(n < 256 ? n : 256)" in src and len(calls) == 12
    seen = {}
    for i, j, _ in calls:
        n = min(64 * (8 - i - j), 256)
        assert (i + j) * 64 + n <= 512 and j * 64 + n <= 512
        for q in range(n // 64):
            seen[(i, j + q)] = seen.get((i, j + q), 0) + 1
    assert seen == {(i, j): 1 for i in range(8) for j in range(8) if i + j <= 7}
    assert [c[2] for c in calls[:2]] == ["accumulate"] * 2 and {c[2] for c in calls[2:]} == {"1u"}
    assert [(c[0], c[1]) for c in calls[:2]] == [(0, 0), (0, 4)]


def test_layout_refuses_lists_shorter_than_their_sequences():
    """A sequence whose own list of pages is too short is refused, although
    another sequence's list is long enough to widen the table."""
    from suf_b200 import attention as at

    for pages in ([[1], [2, 3]], [[], [2]], [[1, 2], [3, 2**31]], [[1, -1], [3]]):
        with pytest.raises(ValueError, match="pages"):
            at.AttnLayout(_Ctx, [1, 1], [20, 10], pages, 16, 4, 2)


@pytest.mark.parametrize("which", ["scores", "values"])
def test_an_empty_tile_list_is_refused(host, which):
    """A list without entries would be a launch without blocks."""
    from suf_b200 import _lib

    assert _attn(host, which, _seqs(**PTRS, d_tiles=P16, n_tiles=0)) == _lib.ERR_INVALID
    assert _attn(host, which, _seqs(**PTRS, d_tiles=P16, n_tiles=1)) == _lib.ERR_UNSUPPORTED
    assert b"host-only" in _lib.lib().sufb200_last_error()


@pytest.mark.parametrize("which", ["scores", "values"])
def test_grids_past_31_bits_are_refused(host, which):
    """Few tokens of very many heads: row tiles times key heads count the grid."""
    from suf_b200 import _lib

    wide = dict(batch=1, tokens=63, max_q=1, min_q=1, kv_heads=2**15)
    assert _attn(host, which, _seqs(**PTRS, **{**wide, "q_heads": 2**20})) == _lib.ERR_UNSUPPORTED
    assert b"host-only" in _lib.lib().sufb200_last_error()
    assert _attn(host, which, _seqs(**PTRS, **{**wide, "q_heads": 2**31 - 2**15})) == _lib.ERR_UNSUPPORTED
    assert b"too many" in _lib.lib().sufb200_last_error()


def test_rowmax_refuses_rows_whose_steps_pass_32_bits(host):
    """Threads step through a row by up to 2^22 words past its end in 32-bit
    places: rows stop at 2^30 words."""
    from suf_b200 import _lib
    from suf_b200 import attention as at

    L, r, g = _lib.lib(), (C.c_uint64 * 2)(1, 2), _arr(P16, P16)
    for w, said in [(2**30, b"host-only"), (2**30 + 1, b"2^30")]:
        assert L.sufb200_rowmax_open_pair(host, g, 1, w, P16, P16, r, P16, None) == _lib.ERR_UNSUPPORTED
        assert said in L.sufb200_last_error()
        assert L.sufb200_rowmax_round_pair(host, g, g, 1, w, P16, P16, P16, r, g, P16, None) == _lib.ERR_UNSUPPORTED
        assert said in L.sufb200_last_error()
        assert L.sufb200_maxdiff_ragged_pair(host, g, g, 1, w, P16, P16, g, None) == _lib.ERR_UNSUPPORTED
        assert said in L.sufb200_last_error()
    for lens in ([2**30 + 1], [3, -1], [2**30, 2**30]):
        with pytest.raises(ValueError, match="row lengths"):
            at.RowMaxPlan(_Ctx, lens)


def test_the_appends_packed_arguments_are_the_structs():
    """What the wrapper packs in one piece lies where the struct's fields are."""
    from suf_b200 import attention as at
    from suf_b200._lib import RopeAppend

    args = RopeAppend()
    at._ROPE_FRONT.pack_into(args, 0, *range(1, 13), *range(13, 20))
    assert at._ROPE_FRONT.size == RopeAppend.d_ek.offset
    assert [v for f in (args.d_q, args.d_k, args.d_v) for v in f] == list(range(1, 7))
    assert [args.q_ts, args.q_hs, args.k_ts, args.k_hs, args.v_ts, args.v_hs] == list(range(7, 13))
    assert [args.d_positions, args.d_slots, args.d_cos, args.d_sin] == list(range(13, 17))
    assert list(args.d_a) == [17, 18] and args.d_dq == 19


def test_sizes_past_32_bits_are_refused():
    """Sizes the entry points hold in 32 bits: refused, not cut off."""
    import types

    import torch

    from suf_b200 import attention as at

    for kw in (dict(q_heads=2**32 + 4), dict(page_size=2**32 + 16)):
        with pytest.raises(ValueError, match="multiple of key heads"):
            at.AttnLayout(_Ctx, **{**dict(q_lens=[1], ctx_lens=[3], block_table=[[0]], page_size=16, q_heads=4,
                                          kv_heads=2), **kw})
    k = (torch.zeros(1, 1, 2, dtype=torch.int64).expand(2**32 + 1, 1, 2),) * 2
    cache = types.SimpleNamespace(device=0, kv_heads=1, head_dim=2)
    with pytest.raises(ValueError, match="2\\^31 tokens"):
        at.rope_append_pair(_Ctx, None, k, k, None, None, None, None, None, None, cache)


def test_plans_of_another_device_are_refused():
    """Layouts, row max plans, truncation bundles and caches hold addresses of the
    device they were made on: a context of another one takes none of them."""
    import types

    from suf_b200 import attention as at

    def made(cls, **kw):
        x = cls.__new__(cls)
        x.__dict__.update(device=1, **kw)
        return x

    layout = made(at.AttnLayout, tokens=1, packed=1, q_heads=1, kv_heads=1, page_size=1)
    plan = made(at.RowMaxPlan, rows=1, rounds=1, pairs=[1], values=[2, 1], widths=[2, 1])
    trunc, cache = made(at.TruncPair, frac_bits=12), made(at.ShareCache, kv_heads=1, page_size=1, head_dim=4)
    here = types.SimpleNamespace(device=0, kv_heads=1, page_size=1, head_dim=4)
    none = (None, None)
    for said, call in [
            ("layout", lambda: at.attn_scores_pair(_Ctx, None, none, none, (1, 2), None, none, layout)),
            ("layout", lambda: at.attn_values_pair(_Ctx, none, none, none, (1, 2), None, none, layout)),
            ("row max plan", lambda: at.rowmax_open_pair(_Ctx, plan, none, (1, 2))),
            ("row max plan", lambda: at.rowmax_round_pair(_Ctx, plan, 0, none, none)),
            ("row max plan", lambda: at.maxdiff_ragged_pair(_Ctx, plan, none, none)),
            ("truncation bundle", lambda: trunc.eval_pair(_Ctx, None, None, None)),
            ("truncation bundle", lambda: at.rope_append_pair(_Ctx, None, none, none, None, None, None, None, trunc, None,
                                                              here)),
            ("cache", lambda: at.rope_append_pair(_Ctx, None, none, none, None, None, None, None, None, None, cache)),
            ("cache", lambda: at.CachedAttentionPair(_Ctx, cache, layout)),
            ("layout", lambda: at.CachedAttentionPair(_Ctx, here, layout))]:
        with pytest.raises(ValueError, match=f"the {said} is on cuda:1, the context on cuda:0"):
            call()


def _layout(q, L, q_heads, kv_heads, causal=True):
    """An AttnLayout's lengths, without its device side."""
    from suf_b200 import attention as at

    lay = at.AttnLayout.__new__(at.AttnLayout)
    lay.q_lens, lay.ctx_lens, lay.causal = np.asarray(q, dtype=np.int64), np.asarray(L, dtype=np.int64), causal
    lay.q_heads, lay.kv_heads = q_heads, kv_heads
    return lay


def test_workspace_places_of_long_sequences(emu):
    """Only sequences with more than eight rows per key head take room, in whole
    key tiles, each disjoint from the others; a batch of long ones alone needs no list."""
    q, L = [2048, 1, 0, 3, 2, 9, 1], [2048, 16384, 777, 300, 500, 0, 0]
    at = _layout(q, L, 8, 2)._plane_keys()  # groups of four: nine rows from three tokens on
    assert at.tolist() == [0, 2048, 2048, 2048, 2048 + 384, 2048 + 384, 2048 + 384, 2048 + 384] and at.dtype == np.int32
    assert _layout([3, 40], [5, 900], 8, 2)._plane_keys() is None
    assert _layout([3, 1], [5, 0], 8, 2)._plane_keys() is None  # the short one has nothing cached
    assert _layout([64] * 40 + [1], [2**26] * 40 + [5], 1, 1)._plane_keys() is None  # past 32 bits
    s = _seqs(plane_keys=2432)
    for p0, p1, n in [(0, 2048, 2048), (2048, 2432, 300), (2432, 2432, 0), (0, 2432, 1)]:
        assert emu.emu_plane_fits(C.byref(s), p0, p1, n)
    for p0, p1, n in [(-128, 128, 5), (0, 128, 129), (64, 256, 5), (2048, 2433, 300), (128, 0, 0), (2**31 - 128, 2**31 - 1, 5),
                      (0, -2**31, 5), (-2**31, 2**31 - 1, 5)]:
        assert not emu.emu_plane_fits(C.byref(s), p0, p1, n), (p0, p1, n)


@pytest.mark.parametrize("which", ["scores", "values"])
def test_wrong_workspace_places_are_refused(host, which):
    from suf_b200 import _lib

    assert _attn(host, which, _seqs(**PTRS, d_plane_keys=P16, plane_keys=256)) == _lib.ERR_UNSUPPORTED
    assert b"host-only" in _lib.lib().sufb200_last_error()
    for kw in [dict(plane_keys=128), dict(d_plane_keys=P16), dict(d_plane_keys=P16, plane_keys=-128),
               dict(d_plane_keys=P16, plane_keys=130), dict(d_plane_keys=P16, plane_keys=2**31)]:
        assert _attn(host, which, _seqs(**PTRS, **kw)) == _lib.ERR_INVALID, kw


def test_long_and_short_sequences_are_bounded_each_for_itself(emu):
    """What deals out the work of whole prompts (the longest of their contexts) and
    of single tokens (the most rows of theirs) comes from those sequences alone,
    and a sequence outside its bound is refused like any other wrong length."""
    q, L = [64, 1, 2, 0, 3], [4096, 65536, 70000, 80000, 100]
    assert _layout(q, L, 32, 8)._bounds() == (4096, 8)
    assert _layout([64, 1, 1], [300, 9000, 5], 32, 8)._bounds() == (300, 4)
    assert _layout([1, 2], [300, 9000], 4, 4)._bounds() == (0, 2) and _layout([20], [9], 4, 4)._bounds() == (9, 0)
    blk = C.c_int64()
    s = _seqs(long_ctx=12, short_rows=4)  # groups of two: long from five tokens on

    def fits(n, ctx):
        return emu.emu_seq_fits(C.byref(s), 0, n, 0, ctx, 0, C.byref(blk))

    assert fits(5, 12) and fits(2, 30) and fits(0, 30) and not fits(5, 13) and not fits(3, 5) and not fits(4, 5)
    s.long_ctx = s.short_rows = 0
    assert fits(5, 13) and fits(3, 5) and fits(4, 30)


@pytest.mark.parametrize("which", ["scores", "values"])
def test_wrong_bounds_of_long_and_short_sequences_are_refused(host, which):
    from suf_b200 import _lib

    for kw in [dict(long_ctx=30), dict(short_rows=8)]:
        assert _attn(host, which, _seqs(**PTRS, **kw)) == _lib.ERR_UNSUPPORTED
        assert b"host-only" in _lib.lib().sufb200_last_error()
    for kw in [dict(long_ctx=31), dict(long_ctx=-1), dict(short_rows=9), dict(short_rows=-1)]:
        assert _attn(host, which, _seqs(**PTRS, **kw)) == _lib.ERR_INVALID, kw


def test_words_that_a_kernel_writes_are_not_read_as_read_only():
    """The second part of wide heads adds to the words it stores: no read-only load
    (ld.global.nc, __ldg) may be given the output."""
    import re

    for name in ("attention.cu", "attention_tc.cu", "attention_rope.cu", "rowmax.cu"):
        src = (ROOT / "suf_b200" / "csrc" / name).read_text()
        assert not re.search(r"\bc\[\d\] = \S*out\b", src), name  # the output under an input's name
        assert not re.search(r"\b(ld_if|ld2_if|ld_stream|__ldg)\(&?(a\.)?(o\.)?out\b", src), name
    plain = re.search(r"uint64_t ld_written_if.*?\n}", (ROOT / "suf_b200" / "csrc" / "attention_tc.cu").read_text(), re.S)
    assert "ld.global.u64" in plain.group() and ".nc" not in plain.group()


@pytest.mark.parametrize("name", ["attention_tc.cu", "ring_gemm_tc.cu"])
def test_barriers_are_fenced_between_their_init_and_the_first_use(name):
    """Copies and commits complete mbarriers through the async proxy: the fence
    that shows it their initialisation stands before the CTA's barrier."""
    src = (ROOT / "suf_b200" / "csrc" / name).read_text()
    parts = src.split("mbar_init(")[1:]
    assert parts
    for part in parts:  # up to the next init, or (the last of a group) up to the barrier
        if "__syncthreads();" in part:
            assert "mbar_init_fence();" in part.split("__syncthreads();")[0]
    fence = (ROOT / "suf_b200" / "csrc" / "umma_i8.cuh").read_text().split("void mbar_init_fence()")[1].split("\n")[0]
    assert "fence.proxy.async.shared::cta" in fence


def test_strides_of_single_entries_do_not_count():
    """One token (or one head) has no step to the next: views that differ in that
    stride alone are taken; others are refused."""
    import types

    import torch

    from suf_b200 import attention as at

    cpu = types.SimpleNamespace(device=-1)  # what get_device() says of CPU tensors
    wide, tight = torch.zeros(3, 50, dtype=torch.int64), torch.zeros(3, 16, dtype=torch.int64)

    def views(tokens, heads, dim=4):
        return tuple(t[:tokens, :heads * dim].unflatten(1, (heads, dim)) for t in (wide, tight))

    assert at._strided(cpu, "k", views(1, 4), (1, 4, 4))[3] == 4
    assert at._strided(cpu, "k", views(1, 1), (1, 1, 4))[:2] == (wide.data_ptr(), tight.data_ptr())
    assert at._strided(cpu, "k", views(0, 4), (0, 4, 4))
    per_head = tuple(torch.zeros(2, 3, n, 4, dtype=torch.int64)[:, :, 0] for n in (1, 2))
    assert at._strided(cpu, "k", tuple(t[:, :1].as_strided((2, 1, 4), (12, s, 1)) for t, s in zip(per_head, (4, 8))),
                       (2, 1, 4))[2] == 12
    for bad, shape in [(views(2, 4), (2, 4, 4)), (per_head, (2, 3, 4))]:
        with pytest.raises(ValueError, match="strides differ"):
            at._strided(cpu, "k", bad, shape)
    with pytest.raises(ValueError, match="adjacent"):
        at._strided(cpu, "k", (torch.zeros(1, 4, 8, dtype=torch.int64)[..., ::2],) * 2, (1, 4, 4))


def test_sizes_past_32_bits_in_any_argument_are_refused(host):
    """Heads, positions, pages and the pages of a sequence are 32-bit fields of the
    C structs: larger sizes are refused, not cut off (tensors without elements
    stand for large ones)."""
    import types

    import torch

    from suf_b200 import _lib
    from suf_b200 import attention as at

    cpu = types.SimpleNamespace(device=-1)
    cache = types.SimpleNamespace(device=-1, kv_heads=1, head_dim=2, _args=_lib.RopeAppend())
    k = (torch.zeros(1, 1, 2, dtype=torch.int64),) * 2
    q = (torch.zeros(1, 1, 2, dtype=torch.int64).expand(1, 2**32 + 4, 2),) * 2
    with pytest.raises(ValueError, match="2\\^31 heads"):
        at.rope_append_pair(cpu, q, k, k, None, None, None, None, None, q, cache)
    table = torch.zeros(2**32 + 5, 0, dtype=torch.int32)
    pos = torch.zeros(1, dtype=torch.int32)
    trunc = types.SimpleNamespace(device=-1, _args=(_lib.TruncDesc * 2)())
    with pytest.raises(ValueError, match="2\\^31 positions"):
        at.rope_append_pair(cpu, None, k, k, pos, pos.long(), table, table, trunc, None, cache)
    lay = at.AttnLayout.__new__(at.AttnLayout)
    lay.device, lay.kv_heads, lay.page_size, lay._seqs, lay.tokens, lay.packed, lay.q_heads = -1, 1, 1, _lib.AttnSeqs(), 0, 0, 1
    pool = torch.zeros(2**32 + 3, 1, 1, 0, dtype=torch.int64)
    with pytest.raises(ValueError, match="2\\^31 pages"):
        at.attn_scores_pair(cpu, None, None, None, (1, 2), pool, (pool, pool), lay)
    L = _lib.lib()
    for heads, said in [((2**31 - 5, 2), b"host-only"), ((2**31 - 4, 2), b"2^31 heads"), ((0, 2**30), b"2^31 heads")]:
        a = _rope(q_heads=heads[0], kv_heads=heads[1])
        assert L.sufb200_rope_append_pair(host, C.byref(a), None) == _lib.ERR_UNSUPPORTED
        assert said in L.sufb200_last_error()


def test_malformed_shares_are_refused_as_such():
    import types

    import torch

    from suf_b200 import attention as at

    cache = types.SimpleNamespace(device=0, kv_heads=1, head_dim=2)
    k = (torch.zeros(1, 1, 2, dtype=torch.int64),) * 2
    for q, kk in [(None, None), (None, ()), (None, 3), ((k[0][0, 0],) * 2, k), (k[0][0], None), ((1, 2), k)]:
        with pytest.raises(ValueError, match="both parties"):
            at.rope_append_pair(_Ctx, q, kk, k, None, None, None, None, None, None, cache)
    for r in (None, 5, (1,), (1, 2, 3)):
        with pytest.raises(ValueError, match="both parties"):
            at._masks(r)


def test_pages_take_fresh_masks_before_they_are_written_again():
    """New masks for the given pages alone, others each time, and nothing left of
    what was opened there."""
    import types

    import torch

    from suf_b200 import attention as at

    cpu = types.SimpleNamespace(device=-1)
    pools = [torch.arange(5 * 2 * 3 * 4).view(5, 2, 3, 4) * (i + 1) + 1 for i in range(6)]
    cache = at.ShareCache.from_tensors(cpu, pools[0], pools[1:3], pools[3], pools[4:6])
    old = [p.clone() for p in pools]
    seen = [p[[1, 3]].clone() for p in pools]
    with pytest.raises(ValueError, match="seed"):
        cache.fresh_masks([1])
    for bad in ([5], [-1, 2], [0, 1 << 40]):
        with pytest.raises(ValueError, match="0 to 4"):
            cache.fresh_masks(bad, seed=1)
    assert all(torch.equal(p, o) for p, o in zip(pools, old))
    for seed in (7, 8):
        cache.fresh_masks([3, 1, 3], seed=seed)
        for i, (p, o) in enumerate(zip(pools, old)):
            assert torch.equal(p[[0, 2, 4]], o[[0, 2, 4]])
            if i in (0, 3):
                assert (p[[1, 3]] == 0).all()
            else:
                assert (p[[1, 3]] != seen[i]).all()
                seen[i] = p[[1, 3]].clone()
    cache._dealer = torch.Generator()  # as the constructor leaves it
    cache.fresh_masks(torch.tensor([2]))
    first = pools[1][2].clone()
    cache.fresh_masks([2])
    assert (pools[1][2] != first).all()
    cache.fresh_masks([])


def test_misaligned_index_arrays_are_refused(host):
    """An array of 4- or 8-byte entries at an odd address would fault the GPU."""
    from suf_b200 import _lib

    L, r, g = _lib.lib(), (C.c_uint64 * 2)(1, 2), _arr(P16, P16)
    P2 = 0x10002
    for which in ("scores", "values"):
        for kw in [dict(d_cu_q=P2), dict(d_cu_ctx=P2), dict(d_block_table=P2), dict(d_row_base=P4),
                   dict(d_tiles=P2, n_tiles=1), dict(d_plane_keys=P2, plane_keys=128)]:
            assert _attn(host, which, _seqs(**{**PTRS, **kw})) == _lib.ERR_INVALID, kw
            assert b"misaligned sequence" in L.sufb200_last_error()
    for kw in [dict(d_slots=P4), dict(d_positions=P2), dict(d_cos=P2), dict(d_sin=P2)]:
        assert L.sufb200_rope_append_pair(host, C.byref(_rope(**kw)), None) == _lib.ERR_INVALID, kw
        assert b"misaligned" in L.sufb200_last_error()
    for a, b, c in [(P2, P16, P16), (P16, P2, P16), (P16, P16, P2)]:
        assert L.sufb200_rowmax_round_pair(host, g, g, 4, 9, a, b, c, r, g, P16, None) == _lib.ERR_INVALID
        if c == P16:
            assert L.sufb200_rowmax_open_pair(host, g, 4, 9, a, b, r, P16, None) == _lib.ERR_INVALID
            assert L.sufb200_maxdiff_ragged_pair(host, g, g, 4, 9, a, b, g, None) == _lib.ERR_INVALID
        assert b"misaligned offsets" in L.sufb200_last_error()
    assert _attn(host, "scores", _seqs(**{**PTRS, "d_cu_q": P4})) == _lib.ERR_UNSUPPORTED  # four bytes will do
