"""What the paged operators' entry points refuse, on the CPU."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch
from torch.autograd import forward_ad

from fade_amd import _lib, rope
from fade_amd.pages import TokenPagePool
from fade_amd.rope import LinearScaled, MRope, Vanilla


def test_forward_mode_is_refused():
    x = torch.ones(3, dtype=torch.float16)
    with forward_ad.dual_level():
        _lib.no_gradient("op", x, None)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for context in (torch.enable_grad(), torch.no_grad()):
            with context, pytest.raises(ValueError, match="op: has no forward-mode derivative"):
                _lib.no_gradient("op", None, x, dual)
        _lib.no_gradient("op", forward_ad.unpack_dual(dual).primal)
    _lib.no_gradient("op", x)


def test_places_of_an_output():
    x = torch.zeros(4, 3, 8)
    rows = torch.zeros(64)
    for t in (x, x.transpose(0, 1), x[::2, :, 1:5], x[:0], x[:1].expand(1, 3, 8), rows.as_strided((2, 3, 8), (24, 8, 1)),
              rows.as_strided((1, 3, 8), (0, 8, 1)), rows.as_strided((2, 1, 8), (9, 3, 1)), x[:0].expand(0, 3, 8)):
        assert _lib.each_once(t), t.stride()
    for t in (x[:1].expand(4, 3, 8), x[:, :1].expand(4, 3, 8), rows.as_strided((3, 3, 8), (4, 12, 1)), rows.as_strided((2, 3, 8), (16, 8, 1))):
        assert not _lib.each_once(t), t.stride()


def test_overlap_of_views():
    """Against the bytes that both tensors hold."""
    rng, room = random.Random(1), torch.zeros(4000, dtype=torch.int16)

    def view():
        while True:
            shape = [rng.choice((1, 2, 3, 5)) for _ in range(rng.randint(1, 4))]
            if rng.random() < 0.6:  # nested strides, in either order, with gaps
                stride, reach = [], 1
                for n in reversed(shape):
                    stride.insert(0, reach)
                    reach *= n + rng.choice((0, 0, 1))
                if rng.random() < 0.5:
                    stride.reverse()
            else:
                stride = [rng.choice((0, 1, 2, 3, 4, 7, 10, 30)) for _ in shape]
            x = room if rng.random() < 0.8 else room.view(torch.int32)
            at = rng.randint(0, 60)
            if at + sum((n - 1) * s for n, s in zip(shape, stride)) < x.numel():
                return x.as_strided(shape, stride, at)

    def held(x):
        at = torch.zeros(x.shape, dtype=torch.int64)
        for d, (n, s) in enumerate(zip(x.shape, x.stride())):
            at += (torch.arange(n) * s).view([-1 if e == d else 1 for e in range(x.dim())])
        size = x.element_size()
        return {(i + x.storage_offset()) * size + e for i in at.flatten().tolist() for e in range(size)}

    seen = set()
    for _ in range(3000):
        a, b = view(), view()
        want = bool(held(a) & held(b))
        assert _lib.overlap(a, b) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        seen.add(want)
    assert len(seen) == 2
    # parts of a projection's output lie between one another
    qkv = torch.zeros(500, 48, 64, dtype=torch.float16)
    q, k = qkv[:, :32], qkv[:, 32:40]
    assert not _lib.overlap(q, k) and _lib.overlap(q, qkv[:, 31:]) and not _lib.overlap(q[:0], q)
    _lib.apart("op", "out", q, q, k=k, none=None)
    for bad, other in ((qkv[:, 1:33], {}), (q.transpose(0, 1)[:, :32].transpose(0, 1), {"k": qkv[:, 31:]})):
        with pytest.raises(ValueError, match="op: out .*overlap"):
            _lib.apart("op", "out", bad, q, **other)


def test_slots_outputs_over_other_memory_are_refused():
    """Every overlap of what is written with anything else of the call, by one byte at least; the entry
    refuses before it launches anything."""
    B, ppr, n, cap = 5, 3, 7, 11
    sizes = dict(lens=4 * B, new_tokens=4 * B, reset=B, table=4 * B * ppr, free_pages=4 * cap, ring=8, table_out=4 * B * ppr, lens_out=4 * B,
                 starts=4 * B + 4, slots=4 * n, positions=4 * n, ring_out=8, status=4)
    written = ("free_pages", "table_out", "lens_out", "starts", "slots", "positions", "ring_out", "status")
    place = {name: (1 << 20) + 4096 * i for i, name in enumerate(sizes)}

    def refused(**at):
        a = _lib.PageSlotsArgs(B, ppr, n, cap)
        for name, x in {**place, **at}.items():
            setattr(a, name, x)
        lib = _lib.load()
        return lib.fade_page_slots(ctypes.byref(a), None) == _lib.FADE_EINVAL and b"overlap" in lib.fade_hip_last_error()

    for name in written:
        for other in sizes:
            if other == name:
                continue
            for at in (place[other], place[other] + sizes[other] - 1 & ~3, place[other] - sizes[name] + 4):
                if (name, other, at) == ("table_out", "table", place["table"]):
                    continue
                assert refused(**{name: at}), (name, other, at - place[other])
    assert refused(table_out=place["table"] + 4)


def test_turns_follow_the_scheme():
    """A scheme whose factor, sections or order are changed turns as a new one does (its tables did already)."""
    s = LinearScaled(theta=1e4, head_dim=64, factor=2.0)
    first = s.turns()
    assert s.turns() is first
    s.factor = 4.0
    assert s.turns() == LinearScaled(theta=1e4, head_dim=64, factor=4.0).turns() != first
    m = MRope(theta=1e6, head_dim=128, mrope_section=[24, 20, 20])
    first = m.turns()
    m.interleaved = True
    assert m.turns() == MRope(theta=1e6, head_dim=128, mrope_section=[24, 20, 20], interleaved=True).turns() != first
    m.mrope_section[:] = [22, 21, 21]
    assert m.turns() == MRope(theta=1e6, head_dim=128, mrope_section=[22, 21, 21], interleaved=True).turns()
    m.mrope_section = [1, 2, 3]
    with pytest.raises(ValueError, match="share out"):
        m.turns()
    m.mrope_section = None
    assert set(m.turns()[1]) == {0} and m.n_axes == 1


def test_first_calls_of_two_threads_share_a_table(monkeypatch):
    """Both launches read the frequencies that stay in memory, where both threads have found none and made some."""

    class Tables(dict):
        def get(self, key):
            return None  # as for a thread that looked before the other stored its own

    monkeypatch.setattr(rope, "_TURN_TABLES", Tables())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    scheme = Vanilla(theta=4321.0, head_dim=32)
    a, b = (rope.rope_args(scheme, 32, torch.device("cpu"), "op") for _ in range(2))
    (kept, turn, axis), = rope._TURN_TABLES.values()
    assert a.turn == b.turn == turn == kept.data_ptr() and a.axis == b.axis == axis == turn + 8 * 16


def test_gather_of_no_tokens():
    pool = TokenPagePool(5, 2, 16, torch.bfloat16, "cpu")
    for B in (0, 2):
        k, v = pool.gather(torch.zeros(B, 3, dtype=torch.int32), 0)  # rows that hold nothing yet
        assert k.shape == v.shape == (B, 2, 0, 16)
        assert pool.gather(torch.zeros(B, 3, dtype=torch.int32), 70)[0].shape == (B, 2, 70, 16)
    with pytest.raises(ValueError, match=">= 0"):
        pool.gather(torch.zeros(2, 3, dtype=torch.int32), -1)


def _workspace(**kw):
    a, nb = _lib.PagedAttnArgs(), ctypes.c_int64(0)
    at = 1 << 20
    base = dict(Hq=32, Hkv=8, D=128, n_pages=9000, pages_per_row=128, q=at, q_st=4096, q_sh=128, out=at, o_st=4096, o_sh=128, k_pages=at,
                v_pages=at, table=at, lens=at, starts=at, sm_scale=0.1)
    for name, x in {**base, **kw}.items():
        setattr(a, name, x)
    assert _lib.load().fade_paged_attn_workspace_bytes(ctypes.byref(a), nb) == 0
    return nb.value


def test_a_chunk_among_decoding_rows_goes_to_the_wide_kernel():
    """The workspace has the wide kernel's sums wherever a row may be longer than a tile of the few-row kernel
    while the others have a token each, whatever the rows' average."""
    for B, Hq in ((2, 32), (16, 32), (64, 32), (64, 8), (200, 32)):
        G = Hq // 8
        step = _workspace(B=B, T=B, Hq=Hq)
        assert _workspace(B=B, T=B - 1 + 16 // G, Hq=Hq) == step or B * G + 16 > 1024
        for T in (B + 16 // G, B - 1 + 193, 16 // G * B, 16 // G * B + 1):
            assert _workspace(B=B, T=T, Hq=Hq) > 2 * step, (B, T, Hq)
    assert _workspace(B=2000, T=2000) > 2 * _workspace(B=2000, T=256)  # rows without tokens: a chunk of 1024 matrix rows at most
