"""The paged 16-bit cache on the CPU: what the C entry points refuse, how the attention's work is
cut (a model of the device code's sums, in its precision), and the schemes' turns."""

from __future__ import annotations

import ctypes
import math
import random
from fractions import Fraction

import numpy as np
import pytest
import torch

from fade_amd import _lib
from fade_amd.pages import TokenPagePool
from fade_amd.rope import LinearScaled, MRope, NoRope, Vanilla, extract_rope_scheme

PI = Fraction("3.14159265358979323846264338327950288419716939937511")


def _call(name, args, *more):
    return getattr(_lib.load(), name)(ctypes.byref(args), *more)


def _attn(**kw):
    a = _lib.PagedAttnArgs()
    base = dict(B=2, T=8, Hq=8, Hkv=2, D=128, n_pages=9, pages_per_row=4, q=1 << 20, q_st=1024, q_sh=128, out=1 << 20, o_st=1024, o_sh=128,
                k_pages=1 << 20, v_pages=1 << 20, table=1 << 20, lens=1 << 20, starts=1 << 20, sm_scale=0.1, mask_mode=0, dtype=0)
    for name, x in {**base, **kw}.items():
        setattr(a, name, x)
    return a


def test_attention_arguments():
    nb = ctypes.c_int64(-1)
    assert _call("fade_paged_attn_workspace_bytes", _attn(), nb) == 0 and nb.value >= 0
    for bad in (dict(D=12), dict(D=264), dict(D=0), dict(B=0), dict(T=-1), dict(Hq=7), dict(Hkv=0), dict(n_pages=0), dict(pages_per_row=0),
                dict(q=None), dict(q=(1 << 20) + 8), dict(q_st=1020), dict(o_sh=126), dict(out=(1 << 20) + 4), dict(k_pages=None),
                dict(v_pages=(1 << 20) + 2), dict(table=None), dict(lens=None), dict(starts=None), dict(sm_scale=0.0), dict(sm_scale=-1.0),
                dict(sm_scale=math.nan), dict(sm_scale=math.inf), dict(mask_mode=1), dict(mask_mode=9), dict(dtype=2), dict(T=1 << 25),
                dict(T=1 << 24, Hq=512, q_st=1 << 16, o_st=1 << 16)):
        a = _attn(**bad)
        assert _call("fade_paged_attn_workspace_bytes", a, nb) == _lib.FADE_EINVAL, bad
        assert _lib.load().fade_hip_last_error()
        assert _call("fade_paged_attn", a, None, 0, None) == _lib.FADE_EINVAL, bad
    a = _attn(pages_per_row=400)  # splits: a workspace, large enough and aligned
    assert _call("fade_paged_attn_workspace_bytes", a, nb) == 0 and nb.value > 0
    for ws, size in ((None, nb.value), (1 << 20, nb.value - 1), ((1 << 20) + 8, nb.value)):
        assert _call("fade_paged_attn", a, ws, size, None) == _lib.FADE_EINVAL
    assert _call("fade_paged_attn", _attn(T=0), None, 0, None) == 0  # no tokens: nothing is launched


def test_slots_and_rope_arguments():
    def slots(**kw):
        a = _lib.PageSlotsArgs()
        at = 1 << 20
        names = [f for f, _ in _lib.PageSlotsArgs._fields_[4:]]
        base = dict(B=2, pages_per_row=3, n_tokens=4, n_free=5, **{f: at + 4096 * i for i, f in enumerate(names)})
        for name, x in {**base, **kw}.items():
            setattr(a, name, x)
        return a

    for bad in (dict(B=0), dict(B=4097), dict(pages_per_row=0), dict(n_tokens=-1), dict(n_free=0), dict(n_free=1 << 26), dict(lens=None),
                dict(table_out=None), dict(slots=None), dict(status=None), dict(lens_out=1 << 20), dict(pages_per_row=1 << 25)):
        assert _call("fade_page_slots", slots(**bad), None) == _lib.FADE_EINVAL, bad

    def rope(**kw):
        a = _lib.RopeArgs()
        for name, x in {**dict(B=1, S=4, D=64, Hq=2, Hkv=0, n_freqs=32, n_axes=1, positions=1 << 20), **kw}.items():
            setattr(a, name, x)
        a.q.src = a.q.dst = 1 << 20
        a.turn = a.axis = 1 << 20
        return a

    for bad in (dict(dtype=3), dict(dtype=-1)):
        assert _call("fade_rope_axes", rope(**bad), None) == _lib.FADE_EINVAL
    for name, x in (("D", 63), ("D", 258), ("n_freqs", 33), ("n_freqs", -1), ("positions", None), ("B", -1), ("B", 1 << 31), ("Hkv", 1), ("n_axes", 0), ("n_axes", 5), ("turn", None), ("axis", None)):
        a = rope()
        setattr(a, name, x)
        assert _call("fade_rope_axes", a, None) == _lib.FADE_EINVAL, name
    a = rope()
    assert _call("fade_paged_append", a, None) == _lib.FADE_EINVAL  # no slots
    a.dtype = 2
    assert _call("fade_paged_append", a, None) == _lib.FADE_EINVAL  # 16-bit pages
    a = rope()
    a.S = 0
    assert _call("fade_rope_axes", a, None) == 0


def _cut(lens, new, G, M, causal, start_cost, pieces, least, grain, snap):
    """What every piece of the line does (walk_start, walk_next and finish of paged_attn.hip), in
    its precision: [(piece, row, tile, first key, last key, first, last)], the cuts {piece: parts}."""
    f = np.float32
    step = -(-M // G) if causal else 0
    base = [max(0, n - k) if causal else n for n, k in zip(lens, new)]
    tiles = [-(-k * G // M) for k in new]

    def cost(b, t):
        return t * (base[b] + start_cost) + step * (t * (t + 1) // 2)

    rows_at = [0]
    for b in range(len(lens)):
        rows_at.append(rows_at[-1] + cost(b, tiles[b]))
    line = rows_at[-1]
    piece = max(least, int(f(f(line) * f(f(1.00002) / f(pieces)))) + 1)
    assert piece * pieces >= line
    done, cuts = [], {}
    snap = min(snap, piece // 3)

    def snapped(x, at, to):
        near = at if x - at < to - x else to
        return near if abs(near - x) <= snap else x

    for w in range(pieces):
        x, end = w * piece, min(w * piece + piece, line)
        tail = None
        while x < end:
            b = next(i for i in range(len(lens)) if rows_at[i] <= x < rows_at[i + 1])
            off = x - rows_at[b]
            a = base[b] + start_cost + 0.5 * step
            t = int(2.0 * off / (a + math.sqrt(a * a + 2.0 * step * off)) if step else off / a)
            t = min(max(t, 0), tiles[b] - 1)
            while t > 0 and cost(b, t) > off:
                t -= 1
            while t + 1 < tiles[b] and cost(b, t + 1) <= off:
                t += 1
            at, c = rows_at[b] + cost(b, t), cost(b, t + 1) - cost(b, t)
            assert at <= x < at + c
            x = snapped(x, at, at + c) if x != at else x
            if x == at + c:
                continue
            to = snapped(end, at, at + c) if end < at + c else end
            if to == at:
                break
            last_row = min((t + 1) * M, new[b] * G) - 1
            seen = max(0, lens[b] - new[b] + last_row // G + 1 if causal else lens[b])
            first, last = x == at, at + c <= to
            lo = min((x - at) // grain * grain, seen)
            hi = seen if last else min((end - at) // grain * grain, seen)
            done.append((w, b, t, lo, hi, first, last))
            tail = (at, c, first, last)
            x = at + c
        if tail and tail[2] and not tail[3]:
            rest = tail[0] + tail[1] - end
            parts = max(int(rest / piece) - 1, 0)
            while piece * parts < rest and parts < pieces:
                parts += 1
            cuts[w] = parts + (parts < 2 or rest - piece * (parts - 1) > snap)
    return tiles, done, cuts


def test_work_is_cut_into_equal_pieces():
    """Every tile's keys are walked once and in order, whole or in a beginning and ends of
    consecutive pieces, which is what the second launch joins."""
    rng = random.Random(0)
    for _ in range(80):
        B, G = rng.choice((1, 2, 5, 64, 65, 150)), rng.choice((1, 2, 4, 7, 20, 71))
        M, grain, start, least, snap = rng.choice(((16, 32, 32, 64, 0), (256, 64, 300, 256, 256), (256, 32, 300, 256, 256)))
        cap = rng.choice((5, 100, 4000)) * 64
        lens = [rng.randint(0, cap) if rng.random() < 0.7 else rng.randint(0, min(cap, 90)) for _ in range(B)]
        new = [rng.choice((0, 1, 1, rng.randint(0, 3000 // G), n)) if n < 20000 else rng.choice((0, 1, 700)) for n in lens]
        pieces, causal = rng.choice((1, 3, 32, 127, 512)), rng.random() < 0.7
        tiles, done, cuts = _cut(lens, new, G, M, causal, start, pieces, least, grain, snap)
        by_tile, slots = {}, set()
        for w, b, t, lo, hi, first, last in done:
            by_tile.setdefault((b, t), []).append((w, lo, hi, first, last))
            if not (first and last):
                assert (w, first) not in slots  # a beginning and an end at most in each piece
                slots.add((w, first))
        assert sorted(by_tile) == [(b, t) for b in range(B) for t in range(tiles[b])]
        for (b, t), parts in by_tile.items():
            last_row = min((t + 1) * M, new[b] * G) - 1
            seen = max(0, lens[b] - new[b] + last_row // G + 1 if causal else lens[b])
            assert parts[0][1] == 0 and parts[0][3] and parts[-1][4] and parts[-1][2] == seen
            assert [p[0] for p in parts] == list(range(parts[0][0], parts[0][0] + len(parts)))
            assert all(p[2] == q[1] for p, q in zip(parts, parts[1:])) and not any(p[3] for p in parts[1:])
            if len(parts) > 1:
                assert cuts.pop(parts[0][0]) == len(parts)
        assert not cuts


def _fractions(scheme):  # (of a turn, in 2^-64)
    turn, axis = scheme.turns()
    return [int.from_bytes(turn[8 * i : 8 * i + 8], "little") for i in range(len(axis))], list(axis)


def test_turns():
    s = Vanilla(theta=1e6, head_dim=128)
    turn, axis = _fractions(s)
    assert axis == [0] * 64 and len(turn) == 64
    for t, f in zip(turn, s.inv_freq().tolist()):
        assert abs(Fraction(t, 2**64) - Fraction(f) / (2 * PI)) <= Fraction(1, 2**65)
    lin = LinearScaled(theta=1e6, head_dim=128, factor=4.0)
    assert all(abs(4 * a - b) <= 2 for a, b in zip(_fractions(lin)[0], turn))
    assert NoRope(head_dim=64).turns() == (b"", b"")


def test_axes_of_the_frequencies():
    m = MRope(theta=1e6, head_dim=128, mrope_section=[16, 24, 24])
    assert m.n_axes == 3 and m.freq_axes() == [0] * 16 + [1] * 24 + [2] * 24
    m = MRope(theta=1e6, head_dim=128, mrope_section=[24, 20, 20], interleaved=True)
    assert m.freq_axes() == [0, 1, 2] * 20 + [0] * 4
    assert MRope(theta=1e6, head_dim=128).freq_axes() == [0] * 64 and MRope(theta=1e6, head_dim=128).n_axes == 1
    for bad in (MRope(theta=1e6, head_dim=128, mrope_section=[16, 24, 23]), MRope(theta=1e6, head_dim=128, mrope_section=[16, 24, 24], interleaved=True)):
        with pytest.raises(ValueError, match="share out"):
            bad.turns()

    class Cfg:
        head_dim, rope_theta, rope_parameters = 256, 1e7, {"mrope_section": [11, 11, 10], "mrope_interleaved": True, "partial_rotary_factor": 0.25}

    s = extract_rope_scheme(Cfg())
    assert isinstance(s, MRope) and s.interleaved and s.n_axes == 3 and len(s.freq_axes()) == 32
    Cfg.rope_parameters = {"mrope_section": [16, 24, 24]}
    assert not extract_rope_scheme(Cfg(), head_dim=128).interleaved


def test_pool():
    pool = TokenPagePool(5, 2, 16, torch.bfloat16, "cpu")
    assert pool.k.shape == (6, 2, 64, 16) and pool.free.tolist() == [1, 2, 3, 4, 5] and pool.ring.tolist() == [0, 5]
    st = pool.start(3, 4)
    assert st.table.shape == (3, 4) and st.lens.tolist() == [0, 0, 0] and st.starts.tolist() == [0, 0, 0, 0]
    pool.k.copy_(torch.randn(pool.k.shape))
    k, v = pool.gather(torch.tensor([[1, 4], [2, 0]], dtype=torch.int32), 70)
    assert k.shape == (2, 2, 70, 16) and torch.equal(k[0, :, 64:], pool.k[4, :, :6]) and not v.any()
    with pytest.raises(ValueError, match="exceeds"):
        pool.gather(torch.zeros(1, 1, dtype=torch.int32), 65)
    for bad in ((0, 1, 16), (1, 0, 16), (1, 1, 12), (1, 1, 264)):
        with pytest.raises(ValueError):
            TokenPagePool(*bad, device="cpu")
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        TokenPagePool(1, 1, 16, torch.float32, "cpu")
