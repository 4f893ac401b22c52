"""Page pool for the INT4 middle tier of ragged caches.

The reference's per-sequence mode zero-pads every row to the longest one
(fade/cache.py:1145-1159); its roadmap item A1 (paged tiers, "FADE v1.0
Release + Future Roadmap.md":41-44) replaces that padding with pages.  Here one
pool of 64-token pages serves every layer of a cache (all layers share the KV
head count and head_dim).  A page holds, for every KV head, the packed K codes,
the packed V codes and the per-token V scales of 64 consecutive middle tokens
of one row: exactly one middle tile of the decode kernel, which reads pages
through a per-row block table (``fade_mid_tier.pages``).  The per-channel K
scales span a row's whole middle tier and stay per row ([B, Hkv, 1, D]),
outside the pool.

Page 0 is all zeros and is never handed out.  Block-table slots past a row's
own pages point at it, so gathering a row's pages back into a padded tensor
gives zeros past the row's tokens, which is what the quantizers write for the
zero-padded rows of the unpaged layout: ``gather(store(x))`` is ``x``.

``TokenPagePool`` holds whole 16-bit rows (a prompt's tokens before the compression,
rows of different lengths) in the same 64-token pages.  Its block tables, slot maps
and free pages stay on the GPU: ``page_slots`` makes them from the rows' token counts
in one launch.

``MiddlePagePool``: pages are allocated and freed on the host (a free list); the copies into and
out of the pool run on the current stream, so a page freed by one
reassignment and reused by the next is overwritten only after every earlier
read of it in stream order.
"""

from __future__ import annotations

import bisect
import ctypes
import operator
from dataclasses import dataclass

import torch
from torch import Tensor

from . import _lib

PAGE_TOKENS = 64
_REQUIRES_GRAD = operator.attrgetter("requires_grad")


class MiddlePagePool:
    """``n_pages`` pages of ``PAGE_TOKENS`` middle tokens for ``n_kv_heads`` heads of
    ``head_dim`` channels (reference INT4 layout: two codes a byte, fp16 V scale per
    token).  Storage: ``k_codes``/``v_codes`` uint8 [n_pages + 1, Hkv, 64, D/2] and
    ``v_scale`` fp16 [n_pages + 1, Hkv, 64, 1]; index 0 is the zero page."""

    def __init__(self, n_pages: int, n_kv_heads: int, head_dim: int, device="cuda") -> None:
        if n_pages < 1 or n_kv_heads < 1 or head_dim < 2 or head_dim % 2:
            raise ValueError(
                f"MiddlePagePool needs n_pages >= 1, n_kv_heads >= 1 and an even head_dim, "
                f"got {n_pages}, {n_kv_heads}, {head_dim}"
            )
        self.n_pages = int(n_pages)
        self.n_kv_heads = int(n_kv_heads)
        self.head_dim = int(head_dim)
        dev = torch.device(device)
        shape = (self.n_pages + 1, self.n_kv_heads, PAGE_TOKENS, self.head_dim // 2)
        self.k_codes = torch.zeros(shape, dtype=torch.uint8, device=dev)
        self.v_codes = torch.zeros(shape, dtype=torch.uint8, device=dev)
        self.v_scale = torch.zeros(shape[:3] + (1,), dtype=torch.float16, device=dev)
        self._free = list(range(self.n_pages, 0, -1))  # pop() hands out the lowest id first
        self._used = bytearray(self.n_pages + 1)

    @property
    def device(self) -> torch.device:
        return self.k_codes.device

    @property
    def n_free(self) -> int:
        return len(self._free)

    @property
    def page_bytes(self) -> int:
        """Bytes one page holds (K codes + V codes + V scales, every KV head)."""
        return self.n_kv_heads * PAGE_TOKENS * (self.head_dim + 2)

    def alloc(self, n: int) -> list[int]:
        if n < 0:
            raise ValueError(f"cannot allocate {n} pages")
        if n > len(self._free):
            raise RuntimeError(f"page pool exhausted: {n} pages requested, {len(self._free)} free of {self.n_pages}")
        ids = [self._free.pop() for _ in range(n)]
        for i in ids:
            self._used[i] = 1
        return ids

    def free(self, ids) -> None:
        ids = [int(i) for i in ids]
        for i in ids:
            if not 1 <= i <= self.n_pages:
                raise ValueError(f"page {i} is not a page of this pool (1..{self.n_pages})")
            if not self._used[i]:
                raise ValueError(f"page {i} is not allocated")
        for i in ids:
            self._used[i] = 0
        self._free.extend(reversed(ids))

    def _check(self, kq: Tensor, vq: Tensor, vs: Tensor) -> None:
        B, H, S = (int(d) for d in kq.shape[:3])
        want = {"k_codes": (kq, (B, H, S, self.head_dim // 2), torch.uint8),
                "v_codes": (vq, (B, H, S, self.head_dim // 2), torch.uint8),
                "v_scale": (vs, (B, H, S, 1), torch.float16)}
        if H != self.n_kv_heads:
            raise ValueError(f"the pool holds {self.n_kv_heads} KV heads, the tier has {H}")
        for name, (t, shape, dt) in want.items():
            if tuple(t.shape) != shape or t.dtype != dt:
                raise ValueError(f"{name}: expected {dt} {shape}, got {t.dtype} {tuple(t.shape)}")
            if t.device != self.device:
                raise ValueError(f"{name} is on {t.device}, the pool on {self.device}")

    def store(self, kq: Tensor, vq: Tensor, vs: Tensor, lens_mid) -> tuple[Tensor, list[list[int]]]:
        """Copy a padded middle tier (``kq``/``vq`` uint8 [B, Hkv, S, D/2], ``vs`` fp16
        [B, Hkv, S, 1]) into newly allocated pages: row b's first ``lens_mid[b]`` tokens
        go to ``ceil(lens_mid[b] / 64)`` pages, the last one zero-filled past them if the
        padded tensors are.  Returns the block table (int32 [B, pages per row] on the
        pool's device, the zero page in unused slots) and each row's page ids."""
        self._check(kq, vq, vs)
        B, _, S = (int(d) for d in kq.shape[:3])
        lens = [int(x) for x in lens_mid]
        if len(lens) != B or any(x < 0 or x > S for x in lens):
            raise ValueError(f"lens_mid must give 0..{S} tokens for each of {B} rows")
        counts = [-(-x // PAGE_TOKENS) for x in lens]
        ids = self.alloc(sum(counts))
        table = torch.zeros(B, max(1, max(counts, default=0)), dtype=torch.int32)
        rows, src_b, src_t, k = [], [], [], 0
        for b, c in enumerate(counts):
            row = ids[k : k + c]
            k += c
            rows.append(row)
            if c:
                table[b, :c] = torch.tensor(row, dtype=torch.int32)
            src_b += [b] * c
            src_t += range(c)
        if ids:
            idx = torch.tensor([ids, src_b, src_t], dtype=torch.long)
            if self.device.type != "cpu":
                idx = idx.pin_memory().to(self.device, non_blocking=True)
            dst, sb, stile = idx[0], idx[1], idx[2]
            pad = -(-S // PAGE_TOKENS) * PAGE_TOKENS - S
            for pool, x in ((self.k_codes, kq), (self.v_codes, vq), (self.v_scale, vs)):
                xp = torch.nn.functional.pad(x, (0, 0, 0, pad)) if pad else x
                tiles = xp.reshape(B, self.n_kv_heads, -1, PAGE_TOKENS, x.shape[-1])
                pool[dst] = tiles[sb, :, stile]  # [n, Hkv, 64, W]
        if self.device.type != "cpu":
            table = table.pin_memory().to(self.device, non_blocking=True)
        return table, rows

    def gather(self, table: Tensor, length: int) -> tuple[Tensor, Tensor, Tensor]:
        """The padded middle tier [B, Hkv, length, ...] (K codes, V codes, V scales) a
        block table describes; ``length`` <= pages per row * 64."""
        B, ppr = (int(d) for d in table.shape)
        if length > ppr * PAGE_TOKENS:
            raise ValueError(f"length {length} exceeds the table's {ppr} pages per row")
        t = table.long()

        def one(pool: Tensor) -> Tensor:
            x = pool[t]  # [B, ppr, Hkv, 64, W]
            x = x.permute(0, 2, 1, 3, 4).reshape(B, self.n_kv_heads, ppr * PAGE_TOKENS, pool.shape[-1])
            return x[:, :, :length].contiguous()

        return one(self.k_codes), one(self.v_codes), one(self.v_scale)


def _check_status(op: str, texts: dict[int, str], status: Tensor) -> None:
    word = int(status.item())
    if word:
        what = [t for b, t in texts.items() if word & b]
        # bits 8 to 15: of the call that it was to go on from
        what += [f"the call before it was not done ({t})" for b, t in _lib.SLOTS_STATUS.items() if word >> 8 & b]
        raise RuntimeError(f"{op}: {', '.join(what)} (nothing was changed)")


@dataclass
class PageSlots:
    """What ``page_slots`` writes (int32, on the GPU).

    ``table`` [B, pages_per_row]: each row's pages, 0 past them.  ``lens`` [B]: its tokens,
    the new ones included.  ``starts`` [B + 1]: the first of its new tokens among all.
    ``slots`` / ``positions`` [n_tokens]: where each new token goes (64 * page + place in
    it) and its position in the row; -1 and 0 past the last one.  ``ring`` [2]: the first
    free page's place and the number of free pages.  ``status`` [1]: 0, or why nothing
    was done (``check()``): of the call that made this state alone, but ``TokenPagePool.accept``
    carries its step's on.  ``by``: the call that made it."""

    table: Tensor
    lens: Tensor
    starts: Tensor
    slots: Tensor
    positions: Tensor
    ring: Tensor
    status: Tensor
    by: str = "page_slots"

    def check(self) -> "PageSlots":
        """Raise RuntimeError where the call was not done (reads the status: a host synchronization)."""
        _check_status(self.by, _lib.SLOTS_STATUS if self.by == "page_slots" else _lib.FORK_STATUS, self.status)
        return self


def page_slots(
    lens: Tensor,
    new: Tensor,
    table: Tensor,
    free: Tensor,
    ring: Tensor,
    n_tokens: int,
    reset: Tensor | None = None,
    out: PageSlots | None = None,
) -> PageSlots:
    """Block table and slot map of a step, from the rows' token counts, in one launch and
    without a host synchronization.

    Row b holds ``lens[b]`` tokens and gets ``new[b]`` more (int32 [B], B up to 4096);
    with ``reset`` (bool or uint8 [B]) a marked row returns its pages first and starts
    anew.  ``table`` int32 [B, pages_per_row] is the present block table, ``free``
    int32 [n] the ring of free pages, written where pages are returned (those are handed out
    from the next call on), ``ring`` int32 [2] its first entry and count.  ``n_tokens``
    is the size of the slot map: at least the new tokens.  ``out`` takes the results
    (its ``table`` may be ``table`` itself; else memory of their own, which is checked).

    All or nothing: where pages run out, a row's table is too short, ``n_tokens`` is too
    small or a count is impossible, ``status`` says so, the table, the lengths and the
    ring come out as they went in, and the slot map is empty.  The same inputs give the
    same results again, so a captured graph can be replayed on them.
    """
    op = "page_slots"
    _lib.require_gpu(lens, new, table, free, ring, reset, op=op)
    if table.dim() != 2:
        raise ValueError(f"{op}: table must be [B, pages_per_row], got {tuple(table.shape)}")
    B, ppr = table.shape
    n, n_free, i32 = int(n_tokens), free.numel(), torch.int32
    if n < 0:
        raise ValueError(f"{op}: n_tokens must be >= 0, got {n}")
    for name, t, size in (("lens", lens, B), ("new", new, B), ("table", table, B * ppr), ("free", free, n_free), ("ring", ring, 2)):
        if t.dtype is not i32 or t.numel() != size or not t.is_contiguous() or (t.dim() != 1 and t is not table):
            raise ValueError(f"{op}: {name} must be a contiguous int32 tensor of {size} elements, got {t.dtype} {list(t.shape)}")
    if reset is not None and (reset.dtype not in (torch.bool, torch.uint8) or reset.shape != (B,) or not reset.is_contiguous()):
        raise ValueError(f"{op}: reset must be a contiguous bool or uint8 [B={B}], got {reset.dtype} {list(reset.shape)}")
    sizes = (B * ppr, B, B + 1, n, n, 2, 1)
    if out is None:  # (one allocation: the table first, on its alignment)
        buf = table.new_empty(sum(sizes))
        parts = buf.split_with_sizes(sizes)
        out = PageSlots(parts[0].view(B, ppr), *parts[1:])
        at = buf.data_ptr()
        ptrs = [at]
        for size in sizes[:-1]:
            at += 4 * size
            ptrs.append(at)
    else:
        res = (out.table, out.lens, out.starts, out.slots, out.positions, out.ring, out.status)
        for name, t, size in zip(("table", "lens", "starts", "slots", "positions", "ring", "status"), res, sizes):
            if t.dtype is not i32 or t.numel() != size or not t.is_contiguous() or t.device != table.device:
                raise ValueError(f"{op}: out.{name} must be contiguous int32 of {size} elements on {table.device}")
        _lib.written(op, *res)
        ptrs = [t.data_ptr() for t in res]
        out.by = op
    _lib.written(op, free)
    a = _lib.PageSlotsArgs(B, ppr, n, n_free, lens.data_ptr(), new.data_ptr(), _lib.ptr(reset), table.data_ptr(), free.data_ptr(),
                           ring.data_ptr(), *ptrs)
    _lib.launch("fade_page_slots", a, table.device)
    return out


@dataclass
class PageFork:
    """What ``page_fork`` writes (int32, on the GPU).

    ``table`` [R, pages_per_row], ``lens`` [R]: the rows' pages and tokens.  ``copies`` [R, 3]:
    the page that row r goes on from, the page of its own that takes its place, and the tokens
    in it (zeros: no copy), for ``paged_copy``.  ``ring`` [2], ``status`` [1] as in ``PageSlots``."""

    table: Tensor
    lens: Tensor
    copies: Tensor
    ring: Tensor
    status: Tensor

    def check(self) -> "PageFork":
        """Raise RuntimeError where the call was not done (reads the status: a host synchronization)."""
        _check_status("page_fork", _lib.FORK_STATUS, self.status)
        return self


def page_fork(
    lens: Tensor,
    table: Tensor,
    free: Tensor,
    ring: Tensor,
    source: Tensor | None = None,
    keep: Tensor | None = None,
    before: Tensor | None = None,
) -> PageFork:
    """Rows that go on from other rows: samples of one prompt, beams, rows cut back or dropped;
    without a host synchronization.

    Row r of the result holds the first ``keep[r]`` tokens (int32 [R]; default, and where it has
    fewer: all) of row ``source[r]`` (int32 [R], -1: an empty row; default: row r itself) of the B rows
    of ``lens`` [B] and ``table`` [B, pages_per_row] (B, R up to 4096), in the same pages.  The page that a row
    goes on writing, its last one where that is not full, is its own: of the rows that end in one
    page the first keeps it, unless a row holds it as a full one, and the others get a free page,
    listed in ``copies``.  Pages without a row are returned to the ring, in the order of their
    numbers, for the calls after this one: the copies take pages that were free before it (where those
    are too few, rows are dropped by one call and branch in the next).  Holders are counted among
    these rows alone: none of their pages may be held by rows elsewhere, such as a copy of ``lens`` and
    ``table`` that is to be forked again.  ``free`` int32 [n] and ``ring`` [2] as in ``page_slots``; pages are numbered
    1 .. n.  ``page_slots``' ``reset`` returns pages without a look at other rows: rows that may
    share pages are dropped here, as ``source[r] = -1``.

    All or nothing: where free pages run out, or a source, a count or a page is impossible,
    ``status`` says so, row r comes out as row r went in (empty from row B on), without copies.
    ``before`` int32 [1]: the status of the call that made the rows, where that was not looked at: if it
    is not 0, nothing is done either, and ``status`` carries it on.
    The same inputs give the same results again, so a captured graph can be replayed on them."""
    op = "page_fork"
    _lib.require_gpu(lens, table, free, ring, source, keep, before, op=op)
    if table.dim() != 2:
        raise ValueError(f"{op}: table must be [B, pages_per_row], got {tuple(table.shape)}")
    B, ppr = table.shape
    R = B if source is None else source.numel()
    for name, t, size in (("lens", lens, B), ("table", table, B * ppr), ("free", free, free.numel()), ("ring", ring, 2), ("source", source, R), ("keep", keep, R), ("before", before, 1)):
        if t is not None and (t.dtype is not torch.int32 or t.numel() != size or not t.is_contiguous() or (t.dim() != 1 and t is not table and t is not before)):
            raise ValueError(f"{op}: {name} must be a contiguous int32 tensor of {size} elements, got {t.dtype} {list(t.shape)}")
    sizes = (R * ppr, R, 3 * R, 2, 1)
    buf = table.new_empty(sum(sizes))  # (one allocation)
    out, lens_out, copies, ring_out, status = buf.split_with_sizes(sizes)
    at = buf.data_ptr()
    lens_at = at + 4 * R * ppr
    _lib.written(op, free)
    a = _lib.PageForkArgs(B, R, ppr, free.numel(), lens.data_ptr(), _lib.ptr(source), _lib.ptr(keep), table.data_ptr(), free.data_ptr(), ring.data_ptr(),
                          at, lens_at, lens_at + 4 * R, lens_at + 16 * R, lens_at + 16 * R + 8)
    _lib.launch_with_workspace("fade_page_fork_after", a, table.device, _lib.ptr(before))
    return PageFork(out.view(R, ppr), lens_out, copies.view(R, 3), ring_out, status)


class PageLayers:
    """The pages of several layers, checked once: ``pages``, a sequence of tensors
    [n_pages, Hkv, 64, D] (each layer's K and V), fp16 or bf16, alike and contiguous, each with
    memory of its own that stays where it is (no ``resize_`` or ``set_`` of them).  Moves within them
    (``paged_copy``, ``paged_compact``) take all of them in one launch."""

    def __init__(self, pages) -> None:
        op = "PageLayers"
        self.pages = tuple(pages)
        if not self.pages:
            raise ValueError(f"{op}: needs at least one tensor of pages")
        first = self.pages[0]
        for t in self.pages:
            if t.dim() != 4 or t.shape[2] != PAGE_TOKENS or t.shape[0] < 1 or t.shape[1] < 1 or t.shape[3] < 8 or t.shape[3] % 8 or t.shape[3] > 256:
                raise ValueError(f"{op}: pages must be [n_pages, Hkv, {PAGE_TOKENS}, D], D a multiple of 8 up to 256, got {tuple(t.shape)}")
            if t.shape != first.shape or t.dtype != first.dtype or t.dtype not in (torch.float16, torch.bfloat16):
                raise ValueError(f"{op}: pages must all be float16 or all bfloat16 of one shape, got {first.dtype} {tuple(first.shape)} and {t.dtype} {tuple(t.shape)}")
            if not t.is_contiguous() or t.is_neg() or t.data_ptr() % 16:
                raise ValueError(f"{op}: pages must be contiguous and 16-byte aligned")
        _lib.require_gpu(*self.pages, op=op)
        self._starts = sorted(t.data_ptr() for t in self.pages)
        self._bytes = first.nbytes
        if any(y - x < self._bytes for x, y in zip(self._starts, self._starts[1:])):
            raise ValueError(f"{op}: pages overlap in memory")
        self._inference = any(t.is_inference() for t in self.pages)
        self.device = first.device
        self.n_pages, self.n_kv_heads, self.head_dim = int(first.shape[0]), int(first.shape[1]), int(first.shape[3])
        self._pointers = (ctypes.c_void_p * len(self.pages))(*(t.data_ptr() for t in self.pages))
        self.pointers = ctypes.addressof(self._pointers)

    def about_to_write(self, op: str, read: dict[str, Tensor]) -> None:
        """Before a kernel writes the pages: refuses gradients, and the memory of what it reads beside them."""
        pages = self.pages
        if torch.autograd.forward_ad._current_level >= 0 or True in map(_REQUIRES_GRAD, pages):
            _lib.no_gradient(op, *pages)
        for name, t in read.items():
            at = t.data_ptr()
            i = bisect.bisect_left(self._starts, at + t.nbytes)
            if i and self._starts[i - 1] + self._bytes > at and t.numel():
                raise ValueError(f"{op}: {name} lies in the pages' memory")
        if self._inference:
            _lib.written(op, *pages)
        else:
            torch.autograd.graph.increment_version(pages)


class TokenPagePool:
    """``n_pages`` pages of 64 tokens of 16-bit K and V: ``k``, ``v`` [n_pages + 1, Hkv, 64, D]
    of ``dtype`` (page 0 holds no tokens), and the free pages on the GPU.

    One step of a batch: ``state = pool.step(state, new, n_tokens)`` gives every new
    token its slot, ``paged_append`` writes K and V there, ``paged_attention`` reads
    the rows' pages.  ``start`` gives the state of an empty batch.  Several layers share
    one pool's tables by holding tensors like ``k`` and ``v`` of their own.

    Rows branch and shrink: ``fork`` makes a batch whose rows go on from rows of another
    (samples of one prompt, beams; -1 drops a row), ``accept`` keeps the verified path of each
    row's drafted tokens.  Both take ``layers``, the ``PageLayers`` of all layers' pages, where
    there are more than the pool's own ``k`` and ``v``.

    A state that was given to ``step``, ``fork`` or ``accept`` is used up, once that call was done: its
    pages are the new state's, or returned, and the holders of a page are counted among the rows of one
    state alone.  Used once more it would return pages that the new state's rows hold, or go on
    writing one of them.  A prompt that is to be sampled again later stays a row of the batch."""

    def __init__(self, n_pages: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.float16, device="cuda") -> None:
        if n_pages < 1 or n_kv_heads < 1 or head_dim < 8 or head_dim % 8 or head_dim > 256:
            raise ValueError(f"TokenPagePool needs n_pages >= 1, n_kv_heads >= 1 and a head_dim that is a multiple of 8 "
                             f"up to 256, got {n_pages}, {n_kv_heads}, {head_dim}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"TokenPagePool holds float16 or bfloat16, got {dtype}")
        self.n_pages, self.n_kv_heads, self.head_dim = int(n_pages), int(n_kv_heads), int(head_dim)
        shape = (self.n_pages + 1, self.n_kv_heads, PAGE_TOKENS, self.head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.free = torch.arange(1, self.n_pages + 1, dtype=torch.int32, device=device)
        self.ring = torch.tensor([0, self.n_pages], dtype=torch.int32, device=device)
        self._own_layers: PageLayers | None = None
        self._shared = False  # rows may share pages

    @property
    def device(self) -> torch.device:
        return self.k.device

    @property
    def layers(self) -> PageLayers:
        """The pool's own pages, as ``fork`` and ``accept`` take them."""
        if self._own_layers is None or self._own_layers.pages[0] is not self.k or self._own_layers.pages[1] is not self.v:
            self._own_layers = PageLayers((self.k, self.v))
        return self._own_layers

    def clear(self) -> None:
        """All pages free, as in a new pool (the tokens in them stay until they are overwritten), e.g. at the
        end of a batch: no state made so far may be used any more, and ``reset`` is taken again."""
        torch.arange(1, self.n_pages + 1, dtype=torch.int32, device=self.device, out=self.free)
        self.ring = torch.zeros(2, dtype=torch.int32, device=self.device)
        self.ring[1:].fill_(self.n_pages)
        self._shared = False

    def start(self, batch: int, pages_per_row: int) -> PageSlots:
        """The state of ``batch`` empty rows of at most ``pages_per_row`` pages."""
        z = lambda *s: torch.zeros(s, dtype=torch.int32, device=self.device)  # noqa: E731
        return PageSlots(z(batch, pages_per_row), z(batch), z(batch + 1), z(0), z(0), self.ring, z(1))

    def step(self, state: PageSlots, new: Tensor, n_tokens: int, reset: Tensor | None = None) -> PageSlots:
        """``page_slots`` for the next ``new[b]`` tokens of every row; the pool keeps the ring.  After a
        ``fork`` rows may share pages, and finished ones are dropped by ``fork`` too, not by ``reset``,
        until the pool is ``clear``ed."""
        if reset is not None and self._shared:
            raise ValueError("TokenPagePool.step: rows may share pages after fork; drop finished rows with fork (source -1) instead of reset, or clear the pool")
        nxt = page_slots(state.lens, new, state.table, self.free, self.ring, n_tokens, reset=reset)
        self.ring = nxt.ring
        return nxt

    def _all_layers(self, op: str, layers: PageLayers | None) -> PageLayers:
        """The pages to move tokens in: all that the tables may name have to be there (a move outside them is not made)."""
        if layers is None:
            return self.layers
        from .kernels.paged import _layers

        layers = _layers(layers)
        if layers.n_pages <= self.n_pages or layers.device != self.device:
            raise ValueError(f"{op}: layers need the pool's pages 0 .. {self.n_pages} on {self.device}, got {layers.n_pages} on {layers.device}")
        return layers

    def _rows(self, f: PageFork, by: str) -> PageSlots:
        self.ring = f.ring
        z = lambda n: torch.zeros(n, dtype=torch.int32, device=self.device)  # noqa: E731
        return PageSlots(f.table, f.lens, z(f.lens.numel() + 1), z(0), z(0), f.ring, f.status, by)

    def fork(self, state: PageSlots, source: Tensor, keep: Tensor | None = None, layers: PageLayers | None = None) -> PageSlots:
        """The state of rows that go on from ``state``'s (``page_fork``): row r has the first ``keep[r]``
        tokens (default: all) of row ``source[r]``, or none where that is -1.  Rows share full pages; the
        page that each goes on writing is copied in every layer where it would be shared.  Its status is its
        own: a step's is to be checked ahead of it, and its own ahead of the next step."""
        from .kernels.paged import paged_copy

        layers = self._all_layers("TokenPagePool.fork", layers)
        f = page_fork(state.lens, state.table, self.free, self.ring, source=source, keep=keep)
        self._shared = True
        paged_copy(f.copies, layers)
        return self._rows(f, "TokenPagePool.fork")

    def accept(self, state: PageSlots, path: Tensor, counts: Tensor, layers: PageLayers | None = None) -> PageSlots:
        """The state after a step of drafted tokens of which each row keeps those numbered
        ``path[b, :counts[b]]`` (``verify_drafts``): their K and V moved together in every layer,
        the pages behind them returned.  Where the step itself was not done (``state.status``), nothing
        is, and the new state's ``check()`` says so."""
        from .kernels.paged import paged_compact

        kept = paged_compact(path, counts, state.table, state.lens, state.starts, self._all_layers("TokenPagePool.accept", layers))
        f = page_fork(state.lens, state.table, self.free, self.ring, keep=kept, before=state.status)
        return self._rows(f, "TokenPagePool.accept")

    def gather(self, table: Tensor, length: int) -> tuple[Tensor, Tensor]:
        """K and V [B, Hkv, length, D] that a block table describes (what stands in a row's
        pages past its own tokens included), e.g. to compress them."""
        B, ppr = (int(d) for d in table.shape)
        if length > ppr * PAGE_TOKENS:
            raise ValueError(f"length {length} exceeds the table's {ppr} pages per row")
        if length < 0:
            raise ValueError(f"length must be >= 0, got {length}")
        n = -(-length // PAGE_TOKENS)
        pages = table[:, :n].long()

        def one(x: Tensor) -> Tensor:
            return x[pages].permute(0, 2, 1, 3, 4).reshape(B, self.n_kv_heads, n * PAGE_TOKENS, self.head_dim)[:, :, :length].contiguous()

        return one(self.k), one(self.v)


__all__ = ["MiddlePagePool", "PAGE_TOKENS", "PageFork", "PageLayers", "PageSlots", "TokenPagePool", "page_fork", "page_slots"]
