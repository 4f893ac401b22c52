"""Speculative steps and branching rows on the CPU: what the C entry points refuse."""

from __future__ import annotations

import ctypes

from fade_amd import _lib

AT = 1 << 20


def test_fork_behind_an_earlier_call_arguments():
    names = [f for f, _ in _lib.PageForkArgs._fields_[4:]]
    a = _lib.PageForkArgs(2, 3, 4, 9, *(AT + 4096 * i for i in range(len(names))))
    lib = _lib.load()
    for name in ("table_out", "lens_out", "copies", "ring_out", "status", "free_pages"):  # what it writes
        at = getattr(a, name)
        assert lib.fade_page_fork_after(ctypes.byref(a), at, AT, 1 << 20, None) == _lib.FADE_EINVAL
        assert b"before" in lib.fade_hip_last_error()
    assert lib.fade_page_fork_after(None, None, None, 0, None) == _lib.FADE_EINVAL
