"""Append to and attention over a paged 16-bit cache (``TokenPagePool``), rows of any lengths.

The reference keeps every row of a batch at one length (its per-sequence mode
zero-pads, fade/cache.py:1145-1159) and materializes the cache for the model's
attention (fade/cache.py:683-842); paged rows are its roadmap's item A1.  Tokens of
all rows come packed one after the other, [tokens, heads, D], with ``page_slots``'
``starts``, ``slots``, ``lens`` and ``table``.
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence

import torch
from torch import Tensor

from .. import _lib
from ..pages import PAGE_TOKENS, PageLayers
from ..rope import RopeScheme, rope_args
from .tiered_attn import _attn_dtype


def _check_pages(op: str, k_pages: Tensor, v_pages: Tensor, dtype: torch.dtype) -> tuple[int, int, int]:
    """(pages, kv heads, head_dim) of a pool's tensors."""
    if k_pages.dim() != 4 or k_pages.shape[2] != PAGE_TOKENS or v_pages.shape != k_pages.shape:
        raise ValueError(f"{op}: pages must be [n_pages, Hkv, {PAGE_TOKENS}, D], got {tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise ValueError(f"{op}: pages must be {dtype}, got {k_pages.dtype} and {v_pages.dtype}")
    if not k_pages.is_contiguous() or not v_pages.is_contiguous() or k_pages.is_neg() or v_pages.is_neg():
        raise ValueError(f"{op}: pages must be contiguous")
    return int(k_pages.shape[0]), int(k_pages.shape[1]), int(k_pages.shape[3])


def paged_append(
    k: Tensor,
    v: Tensor,
    k_pages: Tensor,
    v_pages: Tensor,
    slots: Tensor,
    q: Tensor | None = None,
    positions: Tensor | None = None,
    scheme: RopeScheme | None = None,
    q_out: Tensor | None = None,
) -> Tensor | None:
    """Write new tokens' K and V into their pages, in one launch with the rotation of K and q.

    ``k``, ``v`` [tokens, Hkv, D] fp16 or bf16 (any strides with a contiguous D axis, e.g.
    parts of one projection's output); ``k_pages``, ``v_pages`` [n_pages, Hkv, 64, D] as
    ``TokenPagePool`` holds them; ``slots`` int32 [tokens] from ``page_slots``, distinct;
    tokens whose slot is -1 (or in page 0, or past the pages) are not written.  With
    ``scheme`` K is rotated at ``positions`` (int [tokens] or [axes, tokens]) as
    ``rope_axes`` does, and so is ``q`` [tokens, Hq, D] where given: its rotation is returned
    (``q_out``, which may be ``q`` or other memory, or a new tensor), for every token.
    ``k`` and ``v`` may be views of pages, as long as none of their tokens is written.
    """
    op = "paged_append"
    _lib.require_gpu(k, v, k_pages, v_pages, slots, q, positions, q_out, op=op)
    _lib.no_gradient(op, k, v, q, k_pages, v_pages, q_out)
    dtc = _attn_dtype(k, op)
    n_pages, Hkv, D = _check_pages(op, k_pages, v_pages, k.dtype)
    T = int(k.shape[0])
    if tuple(k.shape) != (T, Hkv, D) or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{op}: k and v must be {k_pages.dtype} [tokens, {Hkv}, {D}], got {tuple(k.shape)} and {v.dtype} {tuple(v.shape)}")
    if q is not None and (q.dim() != 3 or q.shape[0] != T or q.shape[2] != D or q.dtype != k.dtype):
        raise ValueError(f"{op}: q must be {k.dtype} [{T}, Hq, {D}], got {q.dtype} {tuple(q.shape)}")
    if slots.dtype != torch.int32 or tuple(slots.shape) != (T,) or not slots.is_contiguous():
        raise ValueError(f"{op}: slots must be a contiguous int32 [{T}], got {slots.dtype} {list(slots.shape)}")
    if (scheme is None) != (positions is None):
        raise ValueError(f"{op}: a scheme needs positions, and positions a scheme")
    if scheme is None and q is not None:
        raise ValueError(f"{op}: q is taken to be rotated, which needs a scheme")
    if q_out is not None and (q is None or q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.stride(2) != 1 or q_out.is_neg()
                              or not _lib.each_once(q_out)):
        raise ValueError(f"{op}: q_out must be like q with a contiguous head_dim axis and no row twice")
    if scheme is None:
        a = _lib.RopeArgs()
        a.n_axes = 1
    else:
        a = rope_args(scheme, D, k.device, op)
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{op}: positions must be int32 or int64, got {positions.dtype}")
        if positions.dim() not in (1, 2) or positions.shape[-1] != T or (positions.dim() == 2 and positions.shape[0] not in (1, a.n_axes)):
            raise ValueError(f"{op}: positions must be [{T}] or [{scheme.n_axes}, {T}], got {tuple(positions.shape)}")
        a.positions, a.pos64, a.pos_ss = positions.data_ptr(), int(positions.dtype == torch.int64), positions.stride(-1)
        a.pos_sa = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    a.B, a.S, a.D, a.Hkv, a.dtype = 1, T, D, Hkv, dtc
    a.slots, a.n_pages = slots.data_ptr(), n_pages
    read = []

    def rows(t: Tensor, dst: int, sh: int = 0, ss: int = 0):
        st = t.stride()
        if st[2] != 1 or t.is_neg():
            t = t.resolve_neg().contiguous()
            st = t.stride()
        read.append(t)
        return _lib.RopeRows(t.data_ptr(), dst, 0, st[1], st[0], 0, sh, ss)

    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    if abs(kp - vp) < k_pages.nbytes:
        raise ValueError(f"{op}: k_pages and v_pages overlap in memory")
    given = q_out is not None

    if q is not None:
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)  # (half the time of torch.empty)
        else:
            _lib.written(op, q_out)
        a.Hq, a.q = q.shape[1], rows(q, q_out.data_ptr(), q_out.stride(1), q_out.stride(0))
    a.k, a.v = rows(k, kp), rows(v, vp)
    if given:
        _lib.apart(op, "q_out", q_out, read[0], k=read[1], v=read[2], slots=slots, positions=positions, k_pages=k_pages, v_pages=v_pages)
    _lib.written(op, k_pages, v_pages)
    _lib.launch("fade_paged_append", a, k.device)
    return q_out


def _layers(layers: PageLayers | Sequence[Tensor]) -> PageLayers:
    return layers if isinstance(layers, PageLayers) else PageLayers(layers)


def _counts(op: str, layers: PageLayers, shapes: tuple, tensors: dict[str, Tensor]) -> None:
    for (name, t), shape in zip(tensors.items(), shapes):
        if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{op}: {name} must be a contiguous int32 tensor of shape {list(shape)}, got {t.dtype} {list(t.shape)}")
    _lib.require_gpu(layers.pages[0], *tensors.values(), op=op)
    layers.about_to_write(op, tensors)


def paged_copy(copies: Tensor, layers: PageLayers | Sequence[Tensor]) -> None:
    """The copies that ``page_fork`` lists, made in the K and V pages of every layer by one launch.

    ``copies`` int32 [R, 3]: page, its copy's page, tokens (the first ones of the page, 0 for no
    copy); no page twice among the copies' pages, and none of them copied from.  ``layers``: the
    pages ([n_pages, Hkv, 64, D] each), or better the ``PageLayers`` of them that a program
    keeps.  Copies from or to pages outside the pool (page 0 included) are not made."""
    op = "paged_copy"
    layers = _layers(layers)
    _counts(op, layers, ((copies.shape[0] if copies.dim() else 0, 3),), dict(copies=copies))
    a = _lib.PagedMoveArgs(len(layers.pages), layers.n_pages, layers.n_kv_heads, layers.head_dim, layers.pointers, copies.shape[0], copies.data_ptr())
    _lib.launch("fade_paged_copy", a, layers.device)


def paged_compact(
    path: Tensor,
    counts: Tensor,
    table: Tensor,
    lens: Tensor,
    starts: Tensor,
    layers: PageLayers | Sequence[Tensor],
) -> Tensor:
    """Keep a path of each row's drafted tokens: K and V of its tokens to consecutive places, in
    every layer, by one launch; returns the tokens that each row then has (int32 [B], for
    ``page_fork``'s ``keep``).

    Row b holds ``lens[b]`` tokens in the pages of ``table`` [B, pages_per_row], its last
    ``n = starts[b + 1] - starts[b]`` ones drafted.  ``path`` int32 [B, max_path], max_path up to 1024, numbers the
    ones that stay, rising (``verify_drafts``), ``counts`` [B] how many of them; token
    ``lens - n + path[b, i]`` goes to place ``lens - n + i``.  Numbers outside 0 .. n - 1 move
    nothing.  The drafted tokens' pages must be the row's own, as ``page_fork`` leaves them.
    ``layers``: the pages of all layers, or better the ``PageLayers`` of them."""
    op = "paged_compact"
    layers = _layers(layers)
    if table.dim() != 2 or path.dim() != 2:
        raise ValueError(f"{op}: table must be [B, pages_per_row] and path [B, max_path], got {tuple(table.shape)} and {tuple(path.shape)}")
    (B, ppr), M = table.shape, path.shape[1]
    tensors = dict(path=path, counts=counts, table=table, lens=lens, starts=starts)
    _counts(op, layers, ((B, M), (B,), (B, ppr), (B,), (B + 1,)), tensors)
    kept = torch.empty_like(lens)
    a = _lib.PagedMoveArgs(len(layers.pages), layers.n_pages, layers.n_kv_heads, layers.head_dim, layers.pointers, B, None, M, ppr,
                           path.data_ptr(), counts.data_ptr(), table.data_ptr(), lens.data_ptr(), starts.data_ptr(), kept.data_ptr())
    _lib.launch("fade_paged_compact", a, layers.device)
    return kept


_MASKS = {"bottom_right": _lib.MASK_BOTTOM_RIGHT, "none": _lib.MASK_NONE, "tree": _lib.MASK_TREE}


class PagedAttentionPlan:
    """Validated launch of the paged attention for fixed tensors, whose contents (the
    queries, the pages, the block table, lengths and starts) may change from run to run.
    The plan keeps the workspace of the key splits' sums for runs on the stream that it
    was made on; a run on another stream takes one of its own.  On 256 CUs it has up to
    16 MiB for a decoding step (whose rows all fit 16 matrix rows), with chunks 81 MiB at
    head_dim 128 and 145 MiB at 256, in each plan; ``paged_attention`` takes and returns
    it at every call.

    Args:
        q: [tokens, Hq, D] fp16 or bf16, every row's new tokens one row after the other;
            D a multiple of 8 up to 256, Hq a multiple of Hkv.
        k_pages, v_pages: [n_pages, Hkv, 64, D] of q's dtype (``TokenPagePool``).
        table: int32 [B, pages_per_row], the pages of each row.
        lens: int32 [B], each row's tokens in its pages, the new ones included.
        starts: int32 [B + 1], the first of each row's tokens in q and their end; ``starts[0]`` is 0.
        mask: ``"bottom_right"`` (query i of a row's n sees keys 0 .. lens - n + i),
            ``"none"`` (all lens of them, as a decoder's queries see an encoder's states) or
            ``"tree"`` (keys 0 .. lens - n - 1, and of the row's n new tokens those of ``tree``).
        out: like q, contiguous along D, q itself or other memory; rows at and past ``starts[B]``
            are left as they are.  Default: a new tensor, zeros there.
        tree: with the mask ``"tree"``: int32 [tokens, words], for each new token the row's new
            tokens that it sees, number j as bit j % 32 of word j / 32 (``draft_tree``'s ``bits``, or
            any other mask; tokens past the words are not seen).

    A query that sees no key, or none with a score over -inf, gets zeros; a NaN or an infinity
    in a value reaches the queries that see its key and no others.  Probabilities times
    values are added up in fp32 before the division, so bf16 values must stay under
    2^120 / tokens.  Lengths, starts and pages are read on the
    GPU and kept inside the tensors there: tokens past a row's table do not count, and
    a page id outside the pool reads page 0."""

    def __init__(
        self,
        q: Tensor,
        k_pages: Tensor,
        v_pages: Tensor,
        table: Tensor,
        lens: Tensor,
        starts: Tensor,
        sm_scale: float | None = None,
        mask: str = "bottom_right",
        out: Tensor | None = None,
        tree: Tensor | None = None,
    ) -> None:
        op = "paged_attention"
        if q.dim() != 3:
            raise ValueError(f"{op}: q must be [tokens, Hq, D], got {tuple(q.shape)}")
        if mask not in _MASKS:
            raise ValueError(f"{op}: mask must be one of {sorted(_MASKS)}, got {mask!r}")
        if (tree is None) != (mask != "tree"):
            raise ValueError(f'{op}: the mask "tree" needs tree, and tree that mask')
        _lib.require_gpu(q, k_pages, v_pages, table, lens, starts, out, tree, op=op)
        _lib.no_gradient(op, q, k_pages, v_pages, out)
        dtc = _attn_dtype(q, op)
        n_pages, Hkv, D = _check_pages(op, k_pages, v_pages, q.dtype)
        T, Hq = int(q.shape[0]), int(q.shape[1])
        if q.shape[2] != D:
            raise ValueError(f"{op}: q has head_dim {q.shape[2]}, the pages {D}")
        if table.dim() != 2:
            raise ValueError(f"{op}: table must be [B, pages_per_row], got {tuple(table.shape)}")
        B, ppr = int(table.shape[0]), int(table.shape[1])
        for name, t, shape in (("table", table, (B, ppr)), ("lens", lens, (B,)), ("starts", starts, (B + 1,))):
            if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{op}: {name} must be a contiguous int32 tensor of shape {list(shape)}, got {t.dtype} {list(t.shape)}")
        if tree is not None and (tree.dtype != torch.int32 or tree.dim() != 2 or tree.shape[0] != T or tree.shape[1] < 1 or not tree.is_contiguous()):
            raise ValueError(f"{op}: tree must be a contiguous int32 [{T}, words], got {tree.dtype} {list(tree.shape)}")
        # (the stride of an axis of one element is never used, whatever it says)
        q_st, q_sh = q.stride(0) if T > 1 else 0, q.stride(1) if Hq > 1 else 0
        if q.is_neg() or q.stride(2) != 1 or (q_st | q_sh) % 8 or q.data_ptr() % 16:
            raise ValueError(f"{op}: q needs a contiguous head_dim axis and 16-byte aligned rows (make a copy)")
        self._fresh = out is None
        if out is None:
            out = torch.empty(T, Hq, D, dtype=q.dtype, device=q.device)
        o_st, o_sh = out.stride(0) if T > 1 else D, out.stride(1) if Hq > 1 else D
        if out.shape != q.shape or out.dtype != q.dtype or out.is_neg() or out.stride(2) != 1 or (o_st | o_sh) % 4 \
                or not _lib.each_once(out) or out.data_ptr() % 8:
            raise ValueError(f"{op}: out must be {q.dtype} {tuple(q.shape)} with a contiguous head_dim axis, 8-byte aligned rows and no row twice")
        if not self._fresh:
            _lib.apart(op, "out", out, q, k_pages=k_pages, v_pages=v_pages, table=table, lens=lens, starts=starts, tree=tree)
        a = _lib.PagedAttnArgs()
        a.B, a.T, a.Hq, a.Hkv, a.D, a.n_pages, a.pages_per_row = B, T, Hq, Hkv, D, n_pages, ppr
        a.q, a.q_st, a.q_sh = q.data_ptr(), q_st, q_sh
        a.out, a.o_st, a.o_sh = out.data_ptr(), o_st, o_sh
        a.k_pages, a.v_pages = k_pages.data_ptr(), v_pages.data_ptr()
        a.table, a.lens, a.starts = table.data_ptr(), lens.data_ptr(), starts.data_ptr()
        a.sm_scale = float(1.0 / math.sqrt(D) if sm_scale is None else sm_scale)
        a.mask_mode, a.dtype, a.zero_tail = _MASKS[mask], dtc, int(self._fresh)
        if tree is not None:
            a.tree, a.tree_words = tree.data_ptr(), tree.shape[1]
        self._keep = (q, k_pages, v_pages, table, lens, starts, tree)
        self.args, self.out = a, out
        self._argp = ctypes.byref(a)
        nb = ctypes.c_int64(0)
        lib = _lib.load()
        _lib.check(lib.fade_paged_attn_workspace_bytes(self._argp, nb), "fade_paged_attn_workspace_bytes")
        self._fn = lib.fade_paged_attn
        self._ws_stream = _lib.current_stream_handle(q.device)
        self.workspace = _lib.scratch(nb.value, q.device) if nb.value else None

    def run(self, stream: int | None = None) -> Tensor:
        dev = self.out.device
        if dev.index != torch.cuda.current_device():
            with torch.cuda.device(dev):
                return self.run(stream)
        s = _lib.current_stream_handle(dev) if stream is None else stream
        ws = self.workspace
        if ws is not None and s != self._ws_stream:  # not the plan's: overlapping runs, and the plan dropped before this one is done
            ws = _lib.scratch_on(ws.numel(), dev, s)
        _lib.written("paged_attention", self.out)
        _lib.check(self._fn(self._argp, None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), s), "fade_paged_attn")
        return self.out


def paged_attention(
    q: Tensor,
    k_pages: Tensor,
    v_pages: Tensor,
    table: Tensor,
    lens: Tensor,
    starts: Tensor,
    sm_scale: float | None = None,
    mask: str = "bottom_right",
    out: Tensor | None = None,
    tree: Tensor | None = None,
) -> Tensor:
    """Attention of each row's new tokens ``q`` [tokens, Hq, D] over the row's pages;
    returns [tokens, Hq, D] of q's dtype.  See ``PagedAttentionPlan`` for the arguments."""
    return PagedAttentionPlan(q, k_pages, v_pages, table, lens, starts, sm_scale, mask, out, tree).run()


__all__ = ["PagedAttentionPlan", "paged_append", "paged_attention", "paged_compact", "paged_copy"]
