"""Rows of a paged cache that branch and shrink, on the GPU: ``page_fork`` against the rows followed on the host,
``paged_copy`` and ``paged_compact`` against the tokens moved one by one, and a pool's steps with drafted tokens
and beams against rows that never shared a page."""

from __future__ import annotations

import math
import random

import pytest
import torch

from fade_amd import _lib
from fade_amd.kernels import draft_tree, paged_append, paged_attention, paged_compact, paged_copy, verify_drafts
from fade_amd.pages import PAGE_TOKENS, PageLayers, TokenPagePool, page_fork
from fade_amd.rope import Vanilla
from test_gpu_paged import _i32, _starts

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _pg(n):
    return -(-n // PAGE_TOKENS)


# ------------------------------------------------------------------ page_fork
class _Model:
    """Rows, their pages and the ring of free pages on the host."""

    def __init__(self, n_pages, ppr, head=0):
        self.cap, self.ppr, self.head, self.count = n_pages, ppr, head, n_pages
        self.free = [0] * n_pages
        for j in range(n_pages):
            self.free[(head + j) % n_pages] = j + 1
        self.rows, self.lens = [], []

    def take(self):
        x = self.free[self.head]
        self.head, self.count = (self.head + 1) % self.cap, self.count - 1
        return x

    def grow(self, new):
        """Rows' next tokens (page_slots)."""
        for b, n in enumerate(new):
            while _pg(self.lens[b] + n) > len(self.rows[b]):
                self.rows[b].append(self.take())
            self.lens[b] += n

    def fork(self, source, keep):
        lens = [0 if s < 0 else min(self.lens[s], k) for s, k in zip(source, keep)]
        rows = [[] if s < 0 else self.rows[s][: _pg(n)] for s, n in zip(source, lens)]
        holders = {}
        for r, row in enumerate(rows):
            for x in row:
                holders.setdefault(x, []).append(r)
        copies = [[0, 0, 0] for _ in rows]
        ends = [row[-1] if n % PAGE_TOKENS else 0 for row, n in zip(rows, lens)]
        need = []
        for r, x in enumerate(ends):
            if x and not (holders[x][0] == r and all(ends[o] == x for o in holders[x])):
                need.append(r)
        if len(need) > self.count:
            return None
        before = {x for row in self.rows for x in row}
        tail = self.head + self.count
        rows = [list(row) for row in rows]
        for r in need:
            copies[r] = [ends[r], self.take(), lens[r] % PAGE_TOKENS]
            rows[r][-1] = copies[r][1]
        for i, x in enumerate(sorted(before - set(holders))):
            self.free[(tail + i) % self.cap] = x
            self.count += 1
        self.rows, self.lens = rows, lens
        return copies

    def table(self):
        return [row + [0] * (self.ppr - len(row)) for row in self.rows]


def _same(got, m, copies, free, ring):
    assert got.table.tolist() == m.table() and got.lens.tolist() == m.lens and got.copies.tolist() == copies
    assert ring.tolist() == [m.head, m.count] and free.tolist() == m.free and int(got.status) == 0


@pytest.mark.parametrize("B,ppr,pages,seed", [(1, 3, 9, 0), (1, 1, 1, 1), (4, 5, 40, 2), (7, 9, 200, 3), (64, 6, 900, 4), (257, 4, 2500, 5), (300, 300, 60000, 6), (1025, 3, 9000, 7),
                                              (4096, 2, 20000, 8), (5, 700, 20000, 9), (12, 4, 70, 10)])
def test_fork_against_the_host(dev, B, ppr, pages, seed):
    rng = random.Random(seed)
    m = _Model(pages, ppr, head=rng.randrange(pages))
    free = _i32(m.free, dev)
    budget = pages // B - 1
    m.rows, m.lens = [[] for _ in range(B)], [0] * B
    m.grow([rng.choice((0, 1, 63, 64, 65, rng.randint(0, ppr * PAGE_TOKENS))) if budget >= ppr else rng.randint(0, max(0, min(budget, ppr)) * PAGE_TOKENS) for _ in range(B)])
    done = 0
    for step in range(8):
        n = len(m.rows)
        lens, table, ring = _i32(m.lens, dev), _i32(m.table(), dev), _i32([m.head, m.count], dev)
        R = n if step % 3 == 0 else min(4096, max(1, n + rng.randint(-n // 2, 3)))
        source = [rng.choice((rng.randrange(n), rng.randrange(min(n, 3)), r % n, -1 if rng.random() < 0.3 else r % n)) for r in range(R)]
        if step == 3:
            source = list(range(n))  # rows stay, some shorter
            R = n
        keep = [rng.choice((2**31 - 1, 10**6, m.lens[s], m.lens[s] // 64 * 64, rng.randint(0, max(0, m.lens[s])))) if s >= 0 else 5 for s in source]
        free_before = free.clone()
        before = (list(map(list, m.rows)), list(m.lens), m.head, m.count)
        copies = m.fork(source, keep)
        args = (lens, table, free, ring)
        kw = dict(keep=_i32(keep, dev))
        if step != 3:
            kw["source"] = _i32(source, dev)
        got = page_fork(*args, **kw)
        if copies is None:
            assert int(got.status) == 1 and torch.equal(free, free_before) and got.ring.tolist() == ring.tolist() and not got.copies.any()
            assert got.lens.tolist() == (before[1] + [0] * R)[:R]
            assert got.table.tolist() == (table.tolist() + [[0] * ppr] * R)[:R]
            with pytest.raises(RuntimeError, match="nothing was changed"):
                got.check()
            continue
        done += 1
        _same(got.check(), m, copies, free, got.ring)
        again = page_fork(*args, **kw)  # the inputs stand, and give the same results again
        _same(again, m, copies, free, again.ring)
        # rows go on writing: their last pages are their own
        room = [min(ppr * PAGE_TOKENS - L, 70) for L in m.lens]
        new = [rng.randint(0, r) if rng.random() < 0.5 else 0 for r in room]
        if sum(_pg(L + k) - _pg(L) for L, k in zip(m.lens, new)) <= m.count:
            m.grow(new)
        holders = {}
        for r, row in enumerate(m.rows):
            for j, x in enumerate(row):
                holders.setdefault(x, []).append((r, j))
        for r, (row, L) in enumerate(zip(m.rows, m.lens)):
            if L % PAGE_TOKENS:
                assert len(holders[row[-1]]) == 1
    assert done


def test_fork_defaults_and_shrinking(dev):
    """Without source and keep the rows stay; a full page that a shortened row goes on writing is copied, and kept where nobody else holds it."""
    lens, table = _i32([130, 128, 70], dev), _i32([[1, 2, 3], [1, 2, 0], [4, 5, 0]], dev)
    free, ring = _i32([6, 7, 8, 9, 0, 0, 0, 0, 0], dev), _i32([0, 4], dev)
    got = page_fork(lens, table, free, ring).check()
    assert got.table.tolist() == table.tolist() and got.lens.tolist() == lens.tolist() and not got.copies.any() and got.ring.tolist() == [0, 4]
    got = page_fork(lens, table, free, ring, keep=_i32([100, 999, 3], dev)).check()
    assert got.table.tolist() == [[1, 6, 0], [1, 2, 0], [4, 0, 0]] and got.lens.tolist() == [100, 128, 3]
    assert got.copies.tolist() == [[2, 6, 36], [0, 0, 0], [0, 0, 0]] and got.ring.tolist() == [1, 5] and free.tolist() == [6, 7, 8, 9, 3, 5, 0, 0, 0]
    # one row to four, one of them on the original
    got = page_fork(lens, table, free, ring, source=_i32([0, 0, 0, 0], dev)).check()
    assert got.table.tolist() == [[1, 2, 3], [1, 2, 6], [1, 2, 7], [1, 2, 8]] and got.ring.tolist() == [3, 3] and free.tolist()[4:6] == [4, 5]
    # nobody stays
    got = page_fork(lens, table, free, ring, source=_i32([-1], dev)).check()
    assert got.table.tolist() == [[0, 0, 0]] and got.lens.tolist() == [0] and got.ring.tolist() == [0, 9] and free.tolist() == [6, 7, 8, 9, 1, 2, 3, 4, 5]


@pytest.mark.parametrize("bad", [dict(source=[0, 2]), dict(source=[-2, 0]), dict(keep=[5, -1]), dict(lens=[-1, 3]), dict(lens=[3, 193]), dict(table=[[1, 2, 9], [4, 0, 0]]),
                                 dict(table=[[1, -2, 3], [4, 0, 0]]), dict(table=[[0, 2, 3], [4, 0, 0]]), dict(ring=[8, 1]), dict(ring=[-1, 1]), dict(ring=[0, 9]), dict(ring=[0, -1]),
                                 dict(ring=[0, 7], source=[-1, -1])])
def test_fork_impossible_counts(dev, bad):
    free = _i32([5, 6, 7, 8, 0, 0, 0, 0], dev)
    x = {**dict(lens=[130, 3], table=[[1, 2, 3], [4, 0, 0]], ring=[0, 4], source=[1, 0], keep=[9999, 9999]), **bad}
    args = (_i32(x["lens"], dev), _i32(x["table"], dev), free, _i32(x["ring"], dev))
    got = page_fork(*args, source=_i32(x["source"], dev), keep=_i32(x["keep"], dev))
    assert int(got.status) == 8 and got.table.tolist() == x["table"] and got.lens.tolist() == x["lens"] and got.ring.tolist() == x["ring"]
    assert not got.copies.any() and free.tolist() == [5, 6, 7, 8, 0, 0, 0, 0]


def test_fork_refusals(dev):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    ok = dict(lens=z(2), table=z(2, 3), free=z(5), ring=z(2), source=z(4), keep=z(4))
    page_fork(**ok)
    for bad in (dict(lens=z(3)), dict(lens=z(2).long()), dict(table=z(6)), dict(table=z(3, 2).t()), dict(free=z(0)), dict(free=z(5, 1)), dict(ring=z(3)), dict(source=z(3)),
                dict(keep=z(3)), dict(keep=z(4).float()), dict(source=z(2, 2)), dict(source=None), dict(source=z(0), keep=z(0)), dict(source=z(4097), keep=None),
                dict(lens=z(4097), table=z(4097, 1))):
        with pytest.raises(ValueError):
            page_fork(**{**ok, **bad})
    buf = z(9)
    with pytest.raises(ValueError, match="overlap"):
        page_fork(**{**ok, "free": buf[:5], "ring": buf[3:5]})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        page_fork(**{**ok, "lens": ok["lens"].cpu()})


# ------------------------------------------------------------------ moves
@pytest.mark.parametrize("Hkv,D,tensors,dtype", [(1, 8, 1, F16), (8, 128, 2, BF16), (2, 64, 48, F16), (3, 200, 5, BF16), (5, 40, 131, F16), (1, 256, 2, F16)])
def test_copy(dev, Hkv, D, tensors, dtype):
    g = torch.Generator(device=dev).manual_seed(D)
    layers = PageLayers([torch.randn(20, Hkv, PAGE_TOKENS, D, generator=g, device=dev).to(dtype) for _ in range(tensors)])
    want = [x.clone() for x in layers.pages]
    copies = [[3, 7, 1], [0, 0, 0], [3, 8, 63], [5, 9, 64], [6, 10, 17], [0, 11, 5], [4, 0, 5], [99, 12, 5], [4, 99, 5], [-1, 13, 3], [4, 14, -3], [4, 15, 1000]]
    for x in want:
        for src, dst, n in copies[:5] + [[4, 15, 64]]:
            if n:
                x[dst, :, :n] = x[src, :, :n]
    paged_copy(_i32(copies, dev), layers)
    assert all(torch.equal(a, b) for a, b in zip(layers.pages, want))
    paged_copy(_i32([[1, 2, 9]], dev)[:0], layers)
    paged_copy(_i32([[1, 2, 9]], dev), list(layers.pages))
    for x in want:
        x[2, :, :9] = x[1, :, :9]
    assert all(torch.equal(a, b) for a, b in zip(layers.pages, want))


@pytest.mark.parametrize("Hkv,D,tensors,dtype", [(1, 8, 1, F16), (8, 128, 2, BF16), (2, 64, 48, F16), (3, 200, 5, BF16), (5, 40, 131, F16), (16, 256, 2, F16)])
@pytest.mark.parametrize("new", [[1, 5, 0, 12, 64], [300, 2, 0, 1, 70], [1000]])
def test_compact(dev, Hkv, D, tensors, dtype, new):
    rng = random.Random(D + len(new))
    g = torch.Generator(device=dev).manual_seed(D)
    B = len(new)
    lens = [n + rng.randint(0, 200) for n in new]
    ppr = max(map(_pg, lens)) + 1
    ids = rng.sample(range(1, sum(map(_pg, lens)) + 4), sum(map(_pg, lens)))
    table = []
    for L in lens:
        table.append([ids.pop() for _ in range(_pg(L))])
        table[-1] += [0] * (ppr - len(table[-1]))
    n_pages = sum(map(_pg, lens)) + 4
    layers = PageLayers([torch.randn(n_pages, Hkv, PAGE_TOKENS, D, generator=g, device=dev).to(dtype) for _ in range(tensors)])
    want = [x.clone() for x in layers.pages]
    paths = [sorted(rng.sample(range(n), rng.randint(min(n, 1), n))) for n in new]
    M = max(map(len, paths)) + 1
    slot = lambda b, i: (table[b][i // PAGE_TOKENS], i % PAGE_TOKENS)  # noqa: E731
    src, dst = [], []
    for b, path in enumerate(paths):
        for i, x in enumerate(path):
            src.append(slot(b, lens[b] - new[b] + x))
            dst.append(slot(b, lens[b] - new[b] + i))
    (sp, si), (dp, di) = (torch.tensor(x, device=dev).T for x in (src, dst))
    for x in want:
        x[dp, :, di] = x[sp, :, si]
    kept = paged_compact(_i32([p + [7] * (M - len(p)) for p in paths], dev), _i32([len(p) for p in paths], dev), _i32(table, dev), _i32(lens, dev), _i32(_starts(new), dev), layers)
    assert kept.tolist() == [L - n + len(p) for L, n, p in zip(lens, new, paths)]
    assert all(torch.equal(a, b) for a, b in zip(layers.pages, want))


def test_compact_impossible_counts(dev):
    """Numbers outside a row's new tokens, counts past the path, lengths and pages that cannot be: nothing outside the row is touched."""
    x = torch.randn(6, 2, PAGE_TOKENS, 16, device=dev).half()
    layers = PageLayers([x])
    was = x.clone()
    args = lambda path, counts, table, lens, starts: paged_compact(_i32(path, dev), _i32(counts, dev), _i32(table, dev), _i32(lens, dev), _i32(starts, dev), layers).tolist()  # noqa: E731
    assert args([[0, 9, -1]], [3], [[1, 2]], [70], [0, 5]) == [68] and torch.equal(x, was)
    assert args([[0, 1, 2]], [99], [[1, 2]], [70], [0, 5]) == [68] and torch.equal(x, was)
    assert args([[2, 3, 4]], [-4], [[1, 2]], [70], [0, 5]) == [65] and torch.equal(x, was)
    assert args([[2, 3, 4]], [2], [[1, 2]], [3], [0, 5]) == [0] and torch.equal(x, was)
    assert args([[2, 3, 4]], [2], [[1, 2]], [1000], [0, 5]) == [997] and torch.equal(x, was)
    assert args([[2, 3, 4]], [2], [[1, 99]], [70], [0, 5]) == [67] and torch.equal(x, was)
    assert args([[2, 3, 4]], [2], [[1, 0]], [70], [0, 5]) == [67] and torch.equal(x, was)
    assert args([[2, 3, 4]], [2], [[1, 2]], [70], [5, 0]) == [70] and torch.equal(x, was)


def test_compact_lengths_below_zero(dev):
    """A length below zero, the lowest one included, is an empty row: no place is made from it and nothing moves."""
    x = torch.randn(6, 2, PAGE_TOKENS, 16, device=dev).half()
    layers, was = PageLayers([x]), x.clone()
    for low in (-1, -70, -(2**31) + 3, -(2**31)):
        kept = paged_compact(_i32([[0, 2], [1, 2]], dev), _i32([2, 2], dev), _i32([[1, 2], [3, 4]], dev), _i32([low, low], dev), _i32([0, 5, 5], dev), layers)
        assert kept.tolist() == [0, 0] and torch.equal(x, was), low


def test_moves_refusals(dev):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    h = lambda *s: torch.zeros(s, dtype=F16, device=dev)  # noqa: E731
    x, y = h(4, 2, 64, 16), h(4, 2, 64, 16)
    for bad in ([], [x, x], [x, x[1:]], [x, h(5, 2, 64, 16)], [x, y.bfloat16()], [x.float()], [h(4, 2, 32, 16)], [h(4, 2, 64, 12)], [h(4, 2, 64, 264)], [h(4, 2, 16, 64).transpose(2, 3)],
                [h(4 * 2 * 64 * 16 + 1)[1:].view(4, 2, 64, 16)], [h(2, 64, 16)]):
        with pytest.raises(ValueError):
            PageLayers(bad)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PageLayers([x.cpu()])
    layers = PageLayers([x, y])
    paged_copy(z(2, 3), layers)
    for bad in (z(6), z(2, 4), z(2, 3).long(), z(3, 2).t(), y.view(torch.int32).view(-1)[:6].view(2, 3)):
        with pytest.raises(ValueError):
            paged_copy(bad, layers)
    ok = dict(path=z(2, 4), counts=z(2), table=z(2, 3), lens=z(2), starts=z(3), layers=layers)
    paged_compact(**ok)
    for bad in (dict(path=z(3, 4)), dict(path=z(8)), dict(path=z(2, 1025)), dict(path=z(2, 0)), dict(counts=z(3)), dict(table=z(6)), dict(lens=z(2).long()), dict(starts=z(2)),
                dict(counts=y.view(torch.int32).view(-1)[:2])):
        with pytest.raises(ValueError):
            paged_compact(**{**ok, **bad})
    with pytest.raises(ValueError, match="no backward"):
        paged_copy(z(2, 3), [x.clone().requires_grad_()])
    version = x._version
    paged_copy(z(1, 3), layers)
    assert x._version == version + 1


def test_moves_past_32_bits(dev):
    """Pages whose offsets pass 2^32 elements."""
    Hkv, D = 8, 128
    page = Hkv * PAGE_TOKENS * D
    n_pages = 2**32 // page + 6
    x = torch.empty(n_pages, Hkv, PAGE_TOKENS, D, dtype=BF16, device=dev)
    layers = PageLayers([x])
    far = [n_pages - 1, 2**31 // page + 1, n_pages - 3, 2]
    for p in far:
        x[p] = torch.randn(Hkv, PAGE_TOKENS, D, device=dev).bfloat16()
    a, b = x[far[0]].clone(), x[far[1]].clone()
    paged_copy(_i32([[far[0], far[3], 30], [far[1], far[2], 64]], dev), layers)
    assert torch.equal(x[far[3], :, :30], a[:, :30]) and torch.equal(x[far[2]], b)
    kept = paged_compact(_i32([[0, 9, 40]], dev), _i32([3], dev), _i32([[far[1], far[0]]], dev), _i32([100], dev), _i32([0, 50], dev), layers)
    assert kept.tolist() == [53] and torch.equal(x[far[1], :, 50], b[:, 50]) and torch.equal(x[far[1], :, 51], b[:, 59]) and torch.equal(x[far[1], :, 52], a[:, 90 - 64])


# ------------------------------------------------------------------ together
def _append(pool, layers, state, qkv, Hq, Hkv, positions, scheme):
    """New tokens' K and V into every layer's pages, and the last layer's rotated queries."""
    q, k, v = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv], qkv[:, Hq + Hkv :]
    for i in range(0, len(layers.pages), 2):
        qr = paged_append(k * (i + 1), v * (i + 1), layers.pages[i], layers.pages[i + 1], state.slots, q=q, positions=positions, scheme=scheme)
    return qr


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_speculative_steps(dev, dtype):
    """Steps of drafted trees, verified and accepted, leave a cache of the same bits as one that took the accepted
    tokens alone, and their queries see what those of the latter do."""
    rng = random.Random(3)
    g = torch.Generator(device=dev).manual_seed(3)
    B, Hq, Hkv, D, V, n_layers = 4, 8, 2, 64, 500, 3
    scheme = Vanilla(theta=1e4, head_dim=D)
    embed = torch.randn(V, Hq + 2 * Hkv, D, generator=g, device=dev).to(dtype)  # a token's q, k, v

    def make():
        pool = TokenPagePool(60, Hkv, D, dtype, dev)
        more = [torch.zeros_like(pool.k) for _ in range(2 * n_layers - 2)]
        return pool, PageLayers([pool.k, pool.v, *more])

    pool, layers = make()
    plain, plain_layers = make()
    prompt = [70, 3, 128, 64]
    T = sum(prompt)
    ids = torch.randint(V, (T,), generator=g, device=dev)
    states = []
    for p, ls in ((pool, layers), (plain, plain_layers)):
        st = p.step(p.start(B, 8), _i32(prompt, dev), T)
        _append(p, ls, st, embed[ids], Hq, Hkv, st.positions, scheme)
        states.append(st)
    state, other = states
    root = torch.randint(V, (B,), generator=g, device=dev)
    longest = 0
    for step in range(6):
        new = [rng.randint(1, 40) for _ in range(B)]
        trees = [[-1] + [rng.randint(max(0, i - 5), i - 1) for i in range(1, n)] for n in new]
        T = sum(new)
        parents = _i32([p for t in trees for p in t], dev)
        state = pool.step(state, _i32(new, dev), T)
        tree = draft_tree(parents, state.lens, state.starts, max(new))
        draft = torch.softmax(3 * torch.randn(T, V, generator=g, device=dev), -1)
        target = torch.softmax(draft.log() + 0.3 * torch.randn(T, V, generator=g, device=dev), -1)
        up = torch.tensor([_starts(new)[b] + max(p, 0) for b, t in enumerate(trees) for p in t], device=dev)
        tokens = torch.multinomial(draft[up], 1, generator=g)[:, 0]
        tokens[state.starts[:-1].long()] = root
        qr = _append(pool, layers, state, embed[tokens], Hq, Hkv, tree.positions, scheme)
        out = paged_attention(qr, layers.pages[-2], layers.pages[-1], state.table, state.lens, state.starts, mask="tree", tree=tree.bits)
        got = verify_drafts(target, tokens, parents, state.starts, torch.rand(T, generator=g, device=dev), torch.rand(B, generator=g, device=dev), max(new), draft=draft)
        starts, counts, path = state.starts.tolist(), got.counts.tolist(), got.path.tolist()
        longest = max(longest, *counts)
        state = pool.accept(state, got.path, got.counts, layers)
        state.check()
        # the accepted tokens alone, one row after the other
        taken = torch.tensor([starts[b] + i for b in range(B) for i in path[b][: counts[b]]], device=dev)
        other = plain.step(other, got.counts, sum(counts))
        qr = _append(plain, plain_layers, other, embed[tokens[taken]], Hq, Hkv, other.positions, scheme)
        want = paged_attention(qr, plain_layers.pages[-2], plain_layers.pages[-1], other.table, other.lens, other.starts)
        other.check()
        lens = other.lens.tolist()
        assert state.lens.tolist() == lens and pool.ring[1] == plain.ring[1]
        for a, b in zip(layers.pages, plain_layers.pages):
            for r, L in enumerate(lens):
                rows = [x[t[r, : _pg(L)].long()].transpose(1, 2).reshape(-1, Hkv, D)[:L] for x, t in ((a, state.table), (b, other.table))]
                assert torch.equal(*rows), (step, r)
        # the same queries over the same keys, cut elsewhere: within two roundings of the probabilities and the output
        u = torch.finfo(dtype).eps
        big = 2.0 * n_layers * float(embed[:, Hq + Hkv :].abs().max())
        assert bool(((out[taken].double() - want.double()).abs() <= 4 * u * big).all())
        assert got.tokens[torch.arange(B), got.counts.long() - 1].tolist() == got.next.tolist()
        root = got.next
    assert longest > 2


def test_beams(dev):
    """Rows that branch, go on, are dropped and cut back hold the tokens of rows that each have their own pages."""
    rng = random.Random(5)
    g = torch.Generator(device=dev).manual_seed(5)
    Hkv, D, dtype = 2, 32, F16
    pool = TokenPagePool(80, Hkv, D, dtype, dev)
    layers = PageLayers([pool.k, pool.v])
    state, rows = pool.start(2, 6), [[], []]  # rows: the tokens that each holds

    def grow(state, new):
        T = sum(new)
        k = torch.randn(T, Hkv, D, generator=g, device=dev).to(dtype)
        state = pool.step(state, _i32(new, dev), T).check()
        paged_append(k, -k, pool.k, pool.v, state.slots)
        at = 0
        for b, n in enumerate(new):
            rows[b] = rows[b] + list(k[at : at + n].unbind(0))
            at += n
        return state

    state = grow(state, [100, 30])
    for step in range(12):
        n = len(rows)
        source = [rng.randrange(n) if rng.random() < 0.85 else -1 for _ in range(rng.choice((n, 6, 3)))]
        keep = None
        if step % 3 == 2:
            keep = [rng.randint(0, max(1, len(rows[s]))) if s >= 0 and rng.random() < 0.5 else 10**6 for s in source]
        state = pool.fork(state, _i32(source, dev), None if keep is None else _i32(keep, dev), layers if step % 2 else None)
        state.check()
        rows[:] = [list(rows[s])[: keep[r] if keep else None] if s >= 0 else [] for r, s in enumerate(source)]
        state = grow(state, [rng.choice((1, 1, 2, 40)) if len(x) < 300 else 0 for x in rows])
        k, v = pool.gather(state.table, 6 * PAGE_TOKENS)
        assert state.lens.tolist() == [len(x) for x in rows]
        for b, x in enumerate(rows):
            if x:
                want = torch.stack(x, 1)
                assert torch.equal(k[b, :, : len(x)], want) and torch.equal(v[b, :, : len(x)], -want), (step, b)
    held = len(set(state.table.flatten().tolist()) - {0})
    assert pool.ring[1] == 80 - held
    with pytest.raises(ValueError, match="fork"):
        pool.step(state, _i32([0] * len(rows), dev), 0, reset=torch.zeros(len(rows), dtype=torch.bool, device=dev))
    state = pool.fork(state, _i32([-1], dev))
    assert pool.ring[1] == 80


def test_drafted_steps_in_two_graphs(dev):
    """A step of drafted tokens, captured twice and replayed in turn over one pool, with eager steps of another pool
    between: every replay as the eager step."""
    B, Hq, Hkv, D, V, dtype = 3, 4, 2, 64, 300, BF16
    scheme = Vanilla(theta=1e4, head_dim=D)
    g = torch.Generator(device=dev).manual_seed(7)
    new, trees = [6, 1, 9], [[-1, 0, 0, 1, 1, 3], [-1], [-1, 0, 1, 2, 2, 4, 4, 6, 7]]
    T, n = sum(new), _i32([6, 1, 9], dev)
    parents = _i32([p for t in trees for p in t], dev)
    eager, pool = (TokenPagePool(40, Hkv, D, dtype, dev) for _ in range(2))

    def step(p, state, x):
        state = p.step(state, n, T)
        tree = draft_tree(parents, state.lens, state.starts, 9)
        q, k, v = x["qkv"][:, :Hq], x["qkv"][:, Hq : Hq + Hkv], x["qkv"][:, Hq + Hkv :]
        qr = paged_append(k, v, p.k, p.v, state.slots, q=q, positions=tree.positions, scheme=scheme)
        out = paged_attention(qr, p.k, p.v, state.table, state.lens, state.starts, mask="tree", tree=tree.bits)
        got = verify_drafts(x["target"], x["tokens"], parents, state.starts, x["u"], x["f"], 9, draft=x["draft"])
        return p.accept(state, got.path, got.counts), out, got

    def inputs():
        draft = torch.softmax(2 * torch.randn(T, V, generator=g, device=dev), -1)
        return dict(qkv=torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=dev).to(dtype), draft=draft, target=torch.softmax(draft.log() + 0.4 * torch.randn(T, V, generator=g, device=dev), -1),
                    tokens=torch.randint(V, (T,), generator=g, device=dev), u=0.02 * torch.rand(T, generator=g, device=dev), f=torch.rand(B, generator=g, device=dev))

    a = eager.start(B, 6)
    lens, table, ring = a.lens.clone(), a.table.clone(), pool.ring.clone()
    graphs = []
    for _ in range(2):
        x = inputs()

        def run(x=x):
            pool.ring = ring
            st = pool.start(B, 6)
            st.lens, st.table = lens, table
            st, out, got = step(pool, st, x)
            for dst, src in ((lens, st.lens), (table, st.table), (ring, st.ring)):
                dst.copy_(src)
            return st, out, got

        keep = [t.clone() for t in (lens, table, ring, pool.free, pool.k, pool.v)]
        run()
        for t, old in zip((lens, table, ring, pool.free, pool.k, pool.v), keep):
            t.copy_(old)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = run()
        graphs.append((graph, x, res))
    for i in range(8):
        graph, x, (st, out, got) = graphs[i % 2]
        fresh = inputs()
        for name, t in fresh.items():
            x[name].copy_(t)
        a, want, ver = step(eager, a, fresh)
        a.check()
        graph.replay()
        assert int(st.status) == 0 and torch.equal(out, want) and torch.equal(got.path, ver.path) and torch.equal(got.tokens, ver.tokens), i
        assert torch.equal(lens, a.lens) and torch.equal(table, a.table) and torch.equal(ring, a.ring) and torch.equal(pool.free, eager.free)
        torch.cuda.synchronize()
    assert int(lens.sum()) > 8 * B


@pytest.mark.parametrize("B,ppr,pages", [(6, 5, 60), (200, 100, 30000)])
def test_fork_in_two_graphs(dev, B, ppr, pages):
    """Captured in two graphs and replayed in turn, with eager calls between: every replay as the eager call."""
    rng = random.Random(B)
    lens, table, free = _i32([0] * B, dev), torch.zeros(B, ppr, dtype=torch.int32, device=dev), _i32([0] * pages, dev)
    ring, source, keep = _i32([0, 0], dev), _i32([0] * B, dev), _i32([0] * B, dev)
    call = lambda: page_fork(lens, table, free, ring, source=source, keep=keep)  # noqa: E731
    call()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for i in range(6):
        m = _Model(pages, ppr, head=rng.randrange(pages))
        m.rows, m.lens = [[] for _ in range(B)], [0] * B
        m.grow([rng.randint(0, ppr * PAGE_TOKENS // 2) for _ in range(B)])
        src, kept = [rng.randint(-1, B - 1) for _ in range(B)], [rng.choice((10**6, rng.randint(0, 300))) for _ in range(B)]
        for dst, x in ((lens, m.lens), (table, m.table()), (free, m.free), (ring, [m.head, m.count]), (source, src), (keep, kept)):
            dst.copy_(_i32(x, dev))
        was = free.clone()
        copies = m.fork(src, kept)
        graph, out = graphs[i % 2]
        graph.replay()
        _same(out, m, copies, free, out.ring)
        free.copy_(was)
        got = call()
        _same(got, m, copies, free, got.ring)
        torch.cuda.synchronize()


def test_moves_in_inference_mode(dev):
    with torch.inference_mode():
        layers = PageLayers([torch.randn(4, 2, 64, 16, device=dev).half() for _ in range(2)])
        paged_copy(_i32([[1, 2, 9]], dev), layers)
        assert all(torch.equal(x[2, :, :9], x[1, :, :9]) for x in layers.pages)
    with pytest.raises(RuntimeError, match="inference"):
        paged_copy(_i32([[1, 2, 9]], dev), layers)


def test_off_the_current_device(dev, monkeypatch):
    """Every entry point makes its tensors' GPU the current one for its launch (seen on one GPU by its guard)."""
    pool = TokenPagePool(9, 2, 64, F16, dev)
    state = pool.step(pool.start(2, 2), _i32([64, 6], dev), 70)
    parents = _i32([i - 1 for i in range(64)] + [-1, 0, 0, 1, 1, 1], dev)
    target = torch.softmax(torch.randn(70, 33, device=dev), -1)
    tokens = torch.arange(70, device=dev) % 33
    u, f = torch.zeros(70, device=dev), torch.zeros(2, device=dev)

    def calls():
        free = pool.free.clone()
        tree = draft_tree(parents, state.lens, state.starts, 64)
        got = verify_drafts(target, tokens, parents, state.starts, u, f, 64)
        kept = paged_compact(got.path, got.counts, state.table, state.lens, state.starts, pool.layers)
        fork = page_fork(state.lens, state.table, free, pool.ring, keep=kept)
        paged_copy(fork.copies, pool.layers)
        return tree.bits, tree.positions, got.path, got.tokens, kept, fork.table, free

    pool.k.normal_()
    want = calls()
    entered, current = [], [1]

    class Guard:
        def __init__(self, device):
            entered.append(device)

        def __enter__(self):
            current[0] = dev.index or 0

        def __exit__(self, *_):
            current[0] = 1

    with monkeypatch.context() as m:
        m.setattr(_lib, "_GET_DEVICE", lambda: current[0])
        m.setattr(torch.cuda, "current_device", lambda: current[0])
        m.setattr(torch.cuda, "device", Guard)
        got = calls()
    assert len(entered) == 5 and all(torch.equal(a, b) for a, b in zip(got, want))
