"""Every global address that the paged attention forms, on the CPU: a model of its indexing over the pieces that
``test_paged._cut`` gives, against the sizes of the tensors and of the workspace; and the waits that its direct loads carry."""

from __future__ import annotations

import ctypes
import math
import os
import random
import re
import subprocess

import pytest

from fade_amd import _lib
from test_isa_lds_dma_hazards import CSRC, FLAGS, HIPCC, hazards
from test_paged import _cut

PAGE, CUS = 64, 256
HEADER = 16  # bytes of a piece's entry in `cuts`


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _pieces(T, B, G, Hkv, ppr, lm, start, workgroups, least):
    """set_cut of paged_attn.hip."""
    per_tile = -(-(1 << lm) // G)
    line = (T * G // (1 << lm) + min(B, T)) * (ppr * PAGE + start + per_tile)
    return max(1, min(workgroups // Hkv, -(-line // least)))


def _kernels(T, B, G, Hkv, D, ppr, mask):
    """plan_of of paged_attn.hip: (name, log2 of a tile's rows, keys of a step, start cost, pieces, least, snap, its rows)."""
    step = (T - B + 1) * G <= 16 and T * G <= 1024
    per_cu = 8 if D <= 64 else 4 if D <= 128 else 2
    keys = 32 if D > 128 else 64
    few = ("few", 4, 32, 32, _pieces(T, B, G, Hkv, ppr, 4, 32, per_cu * CUS, 64), 64, 0)
    if step:
        return [(*few, lambda n: True)]
    if mask == "tree":
        return [("wide", 8, keys, 300, _pieces(T, B, G, Hkv, ppr, 8, 300, CUS, 128), 128, 128, lambda n: True)]
    wide = ("wide", 8, keys, 300, _pieces(T, B, G, Hkv, ppr, 8, 300, CUS, 256), 256, 256)
    return [(*few, lambda n: n * G <= 16), (*wide, lambda n: n * G > 16)]


def _check(Hq, Hkv, D, lens, new, mask, spare_pages=3):
    """All address ranges of one call; returns how many pieces of tiles were looked at."""
    G, B, T, starts = Hq // Hkv, len(lens), sum(new), _starts(new)
    ppr = max(-(-n // PAGE) for n in lens) + spare_pages
    words = -(-max(new) // 32)
    kernels = _kernels(T, B, G, Hkv, D, ppr, mask)
    rows = sum(p * Hkv * 2 << lm for _, lm, _, _, p, *_ in kernels if p > 1)
    cuts_at = sum(p * Hkv * HEADER for _, _, _, _, p, *_ in kernels)
    if kernels[0][0] == "few" and len(kernels) == 1:  # (the entries of the wide kernel's pieces too, which is not launched)
        cuts_at += _pieces(T, B, G, Hkv, ppr, 8, 300, CUS, 256) * Hkv * HEADER
    a = _lib.PagedAttnArgs()
    at = 1 << 20
    for name, x in dict(B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, n_pages=9, pages_per_row=ppr, q=at, q_st=Hq * D, q_sh=D, out=at, o_st=Hq * D, o_sh=D, k_pages=at, v_pages=at, table=at,
                        lens=at, starts=at, sm_scale=0.1, mask_mode={"tree": 3, "bottom_right": 0}[mask], dtype=0, tree=at, tree_words=words).items():
        setattr(a, name, x)
    nb = ctypes.c_int64(-1)
    assert _lib.load().fade_paged_attn_workspace_bytes(ctypes.byref(a), nb) == 0
    assert nb.value == (cuts_at + rows * (4 * D + 8) if rows else 0)  # the model's pieces are the library's
    seen = 0
    for name, lm, KT, start, pieces, least, snap, takes in kernels:
        mine = [n if takes(n) else 0 for n in new]
        if not any(mine):
            continue
        M = 1 << lm
        tiles, done, cuts = _cut(lens, mine, G, M, mask == "bottom_right", start, pieces, least, KT, snap)
        written = set()
        for w, b, t, lo, hi, first, last in done:
            seen += 1
            assert 0 <= w < pieces and 0 <= lo <= hi <= lens[b] <= ppr * PAGE
            if lo < hi:
                assert lo % KT == 0  # so a step's keys lie in one page: its byte range is the page's
                for key in (lo, lo + (hi - 1 - lo) // KT * KT):
                    assert key % PAGE + KT <= PAGE and b * ppr + key // PAGE < B * ppr
            # matrix rows: queries, tree masks, outputs
            r0, r1 = t * M, min((t + 1) * M, mine[b] * G)
            assert r0 < r1
            qi = (r1 - 1) // G
            assert starts[b] + qi < starts[b + 1] <= T
            if mask == "tree" and lo < hi:
                base = lens[b] - mine[b]
                for key in range(max(lo, (base - 63) // KT * KT) // KT * KT, hi, 32):
                    off = key - base
                    if off > -32 and key < lens[b]:
                        word = [w_ for w_ in (max(off, 0) >> 5, (max(off, 0) >> 5) + 1) if w_ < words]  # (guarded by words)
                        assert all((starts[b] + qi) * words + x < T * words for x in word) and (off < 0 or off >> 5 < words or off >= mine[b])
            if not (first and last):
                assert (w, first) not in written
                written.add((w, first))
                for kvh in (0, Hkv - 1):
                    row = ((w * Hkv + kvh) * 2 + first) * M + (r1 - r0 - 1)
                    assert pieces > 1 and row < pieces * Hkv * 2 * M
        for w, parts in cuts.items():  # the join reads what was written, and nothing else
            assert parts >= 2 and (w, True) in written and all((w + i, False) in written for i in range(1, parts))
        joined = {(w, True) for w in cuts} | {(w + i, False) for w, parts in cuts.items() for i in range(1, parts)}
        assert joined == written
    return seen


def _log_lengths(rng, n, lo, hi):
    out = [hi] if n == 1 else [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    rng.shuffle(out)
    return out


# Hq, Hkv, head_dim, rows, keys from, to, drafted tokens from, to
TREES = [(14, 2, 64, 1, 1000, 1000, 8, 8), (32, 8, 128, 16, 8192, 8192, 8, 16), (28, 4, 128, 61, 190, 32000, 24, 48), (32, 8, 128, 1, 8192, 8192, 16, 16),
         (32, 8, 128, 1, 1000, 1000, 16, 16), (32, 8, 128, 4, 500, 2000, 16, 32), (64, 8, 128, 8, 2000, 6000, 32, 64), (32, 8, 128, 32, 200, 2000, 4, 8),
         (16, 8, 256, 16, 1000, 4000, 12, 24), (28, 4, 128, 16, 100, 3000, 20, 40), *((28, 4, 128, 61, 190, 32000, n, n) for n in (9, 18, 24, 36, 48, 64, 73)),
         *((32, 8, 128, 1, n, n, 8, 8) for n in (8, 56, 120, 248, 504, 2000, 4000))]


@pytest.mark.parametrize("Hq,Hkv,D,B,lo,hi,n0,n1", TREES)
def test_tree_attention_addresses(Hq, Hkv, D, B, lo, hi, n0, n1):
    for seed in range(3):
        rng = random.Random(seed)
        new = [rng.randint(n0, n1) for _ in range(B)]
        lens = [n + k for n, k in zip(_log_lengths(rng, B, lo, hi), new)]
        assert _check(Hq, Hkv, D, lens, new, "tree") >= B
        assert _check(Hq, Hkv, D, lens, new, "bottom_right") >= B


def test_attention_addresses_over_the_range():
    rng = random.Random(1)
    for _ in range(120):
        Hq, Hkv, D = rng.choice(((32, 8, 128), (28, 4, 128), (64, 8, 128), (14, 2, 64), (16, 8, 256), (5, 5, 40), (71, 1, 80), (20, 1, 200)))
        B = int(math.exp(rng.uniform(0, math.log(130))))
        new = [rng.choice((0, 1, 1, rng.randint(1, rng.choice((8, 64, 600))))) for _ in range(B)]
        new[rng.randrange(B)] += 1
        most = rng.choice((1, 100, 3000, 30000))
        lens = [n + rng.randint(0, most) for n in new]
        mask = rng.choice(("tree", "bottom_right"))
        assert _check(Hq, Hkv, D, lens, new, mask, rng.choice((0, 3))) > 0


@pytest.mark.parametrize("DP,NW,KT,NST", [(64, 8, 64, 3), (128, 8, 64, 3), (256, 8, 32, 4)])
def test_wide_kernel_step_loads(DP, NW, KT, NST):
    """A step's direct loads fill its buffer once, from the page's first KT tokens at its place, whatever the head_dim."""
    units, tensor = DP // 8, KT * DP * 2
    per_wave = tensor // 1024 // NW
    exchanged = lambda row, u, v: u ^ ((4 * ((row >> 1) & 1) if v else (row >> 1) & 7) if DP == 64 else (4 * (row & 3) if v else row & 15))  # noqa: E731
    for D in {DP, DP - 8, max(8, DP // 2 + 8), 8}:
        for v in (False, True):
            to, source = set(), set()
            for wave in range(NW):
                for i in range(per_wave):
                    for lane in range(64):
                        pos = 64 * (per_wave * wave + i) + lane
                        row, u = divmod(pos, units)
                        x = exchanged(row, u, v)
                        to.add(1024 * per_wave * wave + 1024 * i + 16 * lane)
                        if 8 * x < D:
                            at = 2 * (row * D + 8 * x)
                            assert at + 16 <= 2 * KT * D
                            source.add(at)
            assert to == set(range(0, tensor, 16)) and source == set(range(0, 2 * KT * D, 16))
    assert 2 * tensor * NST <= 160 * 1024 - 16


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_direct_loads_carry_their_waits(tmp_path):
    """Each direct load follows its own m0 and its own wait states, with nothing between: no path to it, through a branch or from
    a spilled register that is read back, can be shorter."""
    out = tmp_path / "paged_attn.s"
    subprocess.run([HIPCC, *FLAGS, os.path.join(CSRC, "paged_attn.hip"), "-o", str(out)], check=True, capture_output=True, timeout=900)
    asm = out.read_text()
    lines = [s for s in (line.split(";")[0].strip() for line in asm.split("\n")) if s and not s.startswith(".")]
    loads = 0
    for i, s in enumerate(lines):
        if not s.startswith("global_load_lds"):
            continue
        loads += 1
        base = s.split(",")[1].split()[0]
        m0, nop = lines[i - 2], lines[i - 1]
        assert re.match(r"s_mov_b32 m0, s\d+$", m0), (m0, nop, s)
        waits = int(re.match(r"s_nop (\d+)$", nop).group(1)) + 1
        assert waits >= (1 if base == "off" else 4), (m0, nop, s)  # (m0's own write is the fifth)
    assert loads > 100 and hazards(asm)[0] == loads
