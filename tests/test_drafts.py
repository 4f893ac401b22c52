"""Drafted tokens and branching rows on the CPU: what the C entry points refuse, and how the tree attention's work is
cut (a model of the device code's sums, in its precision)."""

from __future__ import annotations

import ctypes
import random

from fade_amd import _lib
from test_paged import _cut

AT = 1 << 20


def _args(kind, base, **kw):
    a = kind()
    for name, x in {**base, **kw}.items():
        setattr(a, name, x)
    return a


def _refused(name, a, *more):
    lib = _lib.load()
    assert getattr(lib, name)(ctypes.byref(a), *more) == _lib.FADE_EINVAL
    assert lib.fade_hip_last_error()


def test_tree_attention_arguments():
    base = dict(B=2, T=8, Hq=8, Hkv=2, D=128, n_pages=9, pages_per_row=4, q=AT, q_st=1024, q_sh=128, out=AT, o_st=1024, o_sh=128, k_pages=AT, v_pages=AT, table=AT,
                lens=AT, starts=AT, sm_scale=0.1, mask_mode=_lib.MASK_TREE, dtype=0, tree=AT, tree_words=2)
    nb = ctypes.c_int64(-1)
    assert _lib.load().fade_paged_attn_workspace_bytes(ctypes.byref(_args(_lib.PagedAttnArgs, base)), nb) == 0
    for bad in (dict(tree=None), dict(tree=AT + 2), dict(tree_words=0), dict(tree_words=-1), dict(tree_words=1 << 21), dict(mask_mode=4)):
        _refused("fade_paged_attn_workspace_bytes", _args(_lib.PagedAttnArgs, base, **bad), nb)
        _refused("fade_paged_attn", _args(_lib.PagedAttnArgs, base, **bad), None, 0, None)
    # no tokens: nothing to look at, nothing is launched
    assert _lib.load().fade_paged_attn(ctypes.byref(_args(_lib.PagedAttnArgs, base, T=0, tree=None)), None, 0, None) == 0
    # the other masks do not look at it
    assert _lib.load().fade_paged_attn_workspace_bytes(ctypes.byref(_args(_lib.PagedAttnArgs, base, mask_mode=0, tree=None, tree_words=0)), nb) == 0


def test_tree_attention_is_cut_into_pieces():
    """Every tile's keys are walked once and in order, whole or in a beginning and ends of consecutive pieces, none
    past the last one, which is what the second launch joins."""
    rng = random.Random(3)
    for _ in range(150):
        B, G, most = rng.choice((1, 2, 16, 61, 130)), rng.choice((1, 4, 7, 8)), rng.choice((20, 1000, 32000))
        lens = [rng.randint(1, most) for _ in range(B)]
        new = [min(n, rng.randint(0, rng.choice((1, 12, 64, 300)))) for n in lens]
        pieces, grain = rng.choice((1, 16, 32, 128, 256)), rng.choice((32, 64))
        tiles, done, cuts = _cut(lens, new, G, 256, False, 300, pieces, 128, grain, 128)
        by_tile = {}
        for w, b, t, lo, hi, first, last in done:
            by_tile.setdefault((b, t), []).append((w, lo, hi, first, last))
        assert sorted(by_tile) == [(b, t) for b in range(B) for t in range(tiles[b])]
        for (b, t), parts in by_tile.items():
            assert parts[0][1] == 0 and parts[0][3] and parts[-1][4] and parts[-1][2] == lens[b]
            assert [p[0] for p in parts] == list(range(parts[0][0], parts[0][0] + len(parts))) and parts[-1][0] < pieces
            assert all(p[2] == q[1] for p, q in zip(parts, parts[1:])) and not any(p[3] for p in parts[1:])
            if len(parts) > 1:
                assert cuts.pop(parts[0][0]) == len(parts)
        assert not cuts


def test_draft_tree_arguments():
    base = dict(B=2, T=8, words=2, parents=AT, lens=AT, starts=AT, bits=AT, depth=AT, positions=AT, status=AT)
    for bad in (dict(B=0), dict(B=1 << 21), dict(T=-1), dict(T=1 << 25), dict(words=0), dict(words=33), dict(parents=None), dict(lens=None), dict(starts=None),
                dict(bits=None), dict(depth=None), dict(positions=None), dict(status=None)):
        _refused("fade_draft_tree", _args(_lib.DraftTreeArgs, base, **bad), None)
    assert _lib.load().fade_draft_tree(None, None) == _lib.FADE_EINVAL


def test_verify_arguments():
    base = dict(B=2, T=8, V=100, max_path=4, target=AT, target_st=100, draft=AT, draft_st=100, tokens=AT, parents=AT, starts=AT, uniforms=AT, final_u=AT, path=AT,
                counts=AT, tokens_out=AT, next=AT, dtype=2, tok64=1)
    nb = ctypes.c_int64(-1)
    assert _lib.load().fade_verify_workspace_bytes(ctypes.byref(_args(_lib.VerifyArgs, base)), nb) == 0 and nb.value >= 0
    for bad in (dict(B=0), dict(B=1 << 21), dict(T=-1), dict(T=1 << 25), dict(V=0), dict(V=1 << 25), dict(max_path=0), dict(max_path=1025), dict(target_st=-1),
                dict(draft_st=-1), dict(dtype=3), dict(dtype=-1), dict(target=None), dict(tokens=None), dict(parents=None), dict(starts=None), dict(uniforms=None),
                dict(final_u=None), dict(path=None), dict(counts=None), dict(tokens_out=None), dict(next=None)):
        _refused("fade_verify_workspace_bytes", _args(_lib.VerifyArgs, base, **bad), nb)
        _refused("fade_verify_drafts", _args(_lib.VerifyArgs, base, **bad), None, 0, None)


def test_page_fork_arguments():
    names = [f for f, _ in _lib.PageForkArgs._fields_[4:]]
    base = dict(B=2, R=3, pages_per_row=4, n_free=9, **{f: AT + 4096 * i for i, f in enumerate(names)})
    nb = ctypes.c_int64(-1)
    assert _lib.load().fade_page_fork_workspace_bytes(ctypes.byref(_args(_lib.PageForkArgs, base)), nb) == 0
    for bad in (dict(B=0), dict(R=0), dict(B=4097), dict(R=4097), dict(pages_per_row=0), dict(pages_per_row=1 << 25), dict(n_free=0), dict(n_free=1 << 26),
                dict(lens=None), dict(table=None), dict(free_pages=None), dict(ring=None), dict(table_out=None), dict(lens_out=None), dict(copies=None),
                dict(ring_out=None), dict(status=None), dict(source=None), dict(table_out=base["table"]), dict(lens_out=base["lens"] + 4),
                dict(ring_out=base["ring"]), dict(copies=base["source"] - 8), dict(free_pages=base["table"] + 28)):
        _refused("fade_page_fork_workspace_bytes", _args(_lib.PageForkArgs, base, **bad), nb)
        _refused("fade_page_fork", _args(_lib.PageForkArgs, base, **bad), AT, 1 << 20, None)


def test_move_arguments():
    pools = (ctypes.c_void_p * 2)(AT, AT + 4096)
    base = dict(n_pools=2, n_pages=5, Hkv=2, D=64, pools=ctypes.addressof(pools), rows=3, copies=AT, max_path=4, pages_per_row=2, path=AT, counts=AT, table=AT,
                lens=AT, starts=AT, kept=AT)
    crooked = (ctypes.c_void_p * 2)(AT, AT + 8)
    empty = (ctypes.c_void_p * 2)(AT, None)
    both = (dict(n_pools=0), dict(n_pools=1 << 16), dict(n_pages=0), dict(n_pages=1 << 31), dict(Hkv=0), dict(D=12), dict(D=264), dict(D=0), dict(pools=None),
            dict(rows=-1), dict(rows=1 << 21), dict(pools=ctypes.addressof(crooked)), dict(pools=ctypes.addressof(empty)))
    for bad in (*both, dict(copies=None)):
        _refused("fade_paged_copy", _args(_lib.PagedMoveArgs, base, **bad), None)
    for bad in (*both, dict(rows=0), dict(max_path=0), dict(max_path=1025), dict(pages_per_row=0), dict(pages_per_row=1 << 25), dict(path=None), dict(counts=None),
                dict(table=None), dict(lens=None), dict(starts=None), dict(kept=None)):
        _refused("fade_paged_compact", _args(_lib.PagedMoveArgs, base, **bad), None)
    assert _lib.load().fade_paged_copy(ctypes.byref(_args(_lib.PagedMoveArgs, base, rows=0)), None) == 0  # nothing to copy: nothing is launched
