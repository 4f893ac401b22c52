"""Speculative steps as a program makes them: trees with filler tokens, steps that could not be done, layers that do not
fit the pool."""

from __future__ import annotations

import random

import pytest
import torch

from fade_amd.kernels import draft_tree, paged_append, paged_compact, paged_copy, verify_drafts
from fade_amd.pages import PageLayers, TokenPagePool, page_fork, page_slots
from fade_amd.rope import Vanilla
from test_gpu_drafts import _drafted, _probs, _tree
from test_gpu_paged import _i32, _starts

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


# ------------------------------------------------------------------ verify_drafts with filler tokens
def _filled(rng, tree, filler):
    """The tree with filler tokens anywhere behind its first one, and each token's number in it."""
    n = len(tree)
    places = sorted(rng.sample(range(1, n + filler), filler))
    number, at = [], 0
    for i in range(n + filler):
        if i not in places:
            number.append(i)
    out = []
    for i in range(n + filler):
        if i in places:
            out.append(rng.choice([number[j] for j in range(n) if number[j] < i]))
        else:
            out.append(-1 if at == 0 else number[tree[at]])
            at += 1
    return out, number


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("V,rows,dtype", [(63, [5, 1, 20], F32), (1001, [9, 70, 4], BF16), (32000, [12], F16), (50000, [12, 6], F32), (151936, [8], BF16)])
def test_filler_tokens_change_nothing(dev, V, rows, dtype, with_draft):
    """Tokens outside the vocabulary (-1 in a tree of a fixed number of tokens) were drawn from nothing: the path and the
    next token are those of the tree without them."""
    torch.manual_seed(V)
    rng = random.Random(V)
    g = torch.Generator(device=dev).manual_seed(V)
    trees = [_tree(rng, n, reach=5) for n in rows]
    target, draft = _probs(g, dev, sum(rows), V, dtype)
    tokens = _drafted(rng, draft, trees)
    filled = [_filled(rng, t, rng.choice((1, 3, 7))) for t in trees]
    many, starts, filled_starts = max(len(f) for f, _ in filled), _starts(rows), _starts([len(f) for f, _ in filled])
    own = torch.tensor([filled_starts[b] + i for b, (_, number) in enumerate(filled) for i in number], device=dev)
    T = filled_starts[-1]
    wide = lambda x, fill: torch.full((T, *x.shape[1:]), fill, dtype=x.dtype, device=dev).index_copy_(0, own, x)  # noqa: E731
    tok = torch.tensor(tokens, device=dev)
    for filler in (-1, V, 2**40, -(2**62)):
        for scale in (1.0, 0.3):
            u, f = scale * torch.rand(sum(rows), generator=g, device=dev), torch.rand(len(rows), generator=g, device=dev)
            want = verify_drafts(target, tok, _i32([p for t in trees for p in t], dev), _i32(starts, dev), u, f, many, draft=draft if with_draft else None)
            got = verify_drafts(wide(target, 0.3), wide(tok, filler), _i32([p for t, _ in filled for p in t], dev), _i32(filled_starts, dev), wide(u, 0.0), f,
                                many, draft=wide(draft, 0.7) if with_draft else None)
            assert torch.equal(got.counts, want.counts) and torch.equal(got.tokens, want.tokens) and torch.equal(got.next, want.next), filler
            for b, (_, number) in enumerate(filled):
                n = int(want.counts[b])
                assert got.path[b, :n].tolist() == [number[i] for i in want.path[b, :n].tolist()] and (got.path[b, n:] == -1).all()


@pytest.mark.parametrize("with_draft", [True, False])
def test_filled_trees_keep_the_targets_distribution(dev, with_draft):
    """The first token that comes out of trees with filler tokens is distributed as the target says."""
    V, B, n = 6, 60000, 5
    g = torch.Generator(device=dev).manual_seed(4)
    p = torch.tensor([0.35, 0.05, 0.25, 0.02, 0.3, 0.03], device=dev)
    q = torch.tensor([0.1, 0.4, 0.2, 0.05, 0.05, 0.2], device=dev)
    parents = _i32([-1, 0, 0, 0, 0] * B, dev)
    starts = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=dev)
    tokens = torch.multinomial(q, B * n, replacement=True, generator=g) if with_draft else torch.tensor([0, 1, 4, 3, 2], device=dev).repeat(B)
    tokens = tokens.view(B, n)
    tokens[:, 1] = -1  # in every row
    tokens[torch.rand(B, generator=g, device=dev) < 0.5, 3] = V  # in half of them
    got = verify_drafts(p.expand(B * n, V), tokens.flatten(), parents, starts, torch.rand(B * n, generator=g, device=dev), torch.rand(B, generator=g, device=dev), 2,
                        draft=q.expand(B * n, V) if with_draft else None)
    share = torch.bincount(got.tokens[:, 0], minlength=V).double() / B
    # six deviations of a share of B drawings
    assert bool(((share - p.double()).abs() <= 6 * (p * (1 - p) / B).sqrt().double()).all()), share.tolist()
    assert 0.2 < float((got.counts == 2).double().mean()) < 0.99


# ------------------------------------------------------------------ steps that could not be done
def _drafted_step(pool, state, new, V, g, dev):
    """A step of a chain of drafted tokens in every row, verified and accepted."""
    T = sum(new)
    parents = _i32([i - 1 for n in new for i in range(n)], dev)
    state = pool.step(state, _i32(new, dev), T)
    tree = draft_tree(parents, state.lens, state.starts, max(new))
    k = torch.randn(T, pool.n_kv_heads, pool.head_dim, generator=g, device=dev).to(pool.k.dtype)
    paged_append(k, k, pool.k, pool.v, state.slots, positions=tree.positions, scheme=Vanilla(theta=1e4, head_dim=pool.head_dim))
    target = torch.softmax(torch.randn(T, V, generator=g, device=dev), -1)
    got = verify_drafts(target, torch.randint(V, (T,), generator=g, device=dev), parents, state.starts, torch.zeros(T, device=dev), torch.rand(len(new), generator=g, device=dev), max(new))
    return state, got, pool.accept(state, got.path, got.counts)


@pytest.mark.parametrize("pages,ppr,B,new,why", [(3, 4, 2, [70, 70], "pages needed than are free"), (9, 1, 2, [60, 70], "pass its table's pages"),
                                                 (20000, 300, 60, [330] * 60, "pages needed than are free")])
def test_accept_carries_a_failed_step_on(dev, pages, ppr, B, new, why):
    """A step that finds no room for its drafted tokens: what accept returns says so, with rows, pages and the ring as
    they were; after it is looked at, a smaller step goes on."""
    g = torch.Generator(device=dev).manual_seed(1)
    pool = TokenPagePool(pages, 1, 8, F16, dev)
    if B == 60:  # (a call of several launches, with most pages in other hands)
        held = torch.tensor([0, 300], dtype=torch.int32, device=dev)
        pool.ring = held
    state = pool.step(pool.start(B, ppr), _i32([5] * B, dev), 5 * B).check()
    k, v = pool.k.normal_(generator=g).clone(), pool.v.normal_(generator=g).clone()
    was = [t.clone() for t in (state.lens, state.table, pool.ring, pool.free)]
    failed, got, after = _drafted_step(pool, state, new, 50, g, dev)
    with pytest.raises(RuntimeError, match=f"^page_slots: .*{why}"):
        failed.check()
    with pytest.raises(RuntimeError, match=f"^TokenPagePool.accept: the call before it was not done .*{why}.*nothing was changed"):
        after.check()
    assert all(torch.equal(a, b) for a, b in zip((after.lens, after.table, pool.ring, pool.free), was)) and torch.equal(after.ring, was[2])
    assert torch.equal(pool.k, k) and torch.equal(pool.v, v) and (got.next == -1).all() and not got.counts.any()
    # and once more, from a state that carries a status on already
    again = pool.accept(after, got.path, got.counts)
    with pytest.raises(RuntimeError, match=f"accept: the call before it .*{why}"):
        again.check()
    _, got, after = _drafted_step(pool, again, [2] * B, 50, g, dev)
    after.check()
    assert after.lens.tolist() == [5 + c for c in got.counts.tolist()] and min(got.counts.tolist()) >= 1


def test_fork_behind_an_earlier_call(dev):
    """page_fork's ``before``: 0 is no matter, anything else leaves all as it is, beside what is wrong with the call itself."""
    lens, table, ring = _i32([70, 3], dev), _i32([[1, 2], [3, 0]], dev), _i32([0, 1], dev)
    free = _i32([4, 0, 0, 0], dev)
    source = _i32([0, 0, -1], dev)
    for before, want in ((0, 0), (1, 0x100), (8, 0x800), (0x200, 0x200), (0x401, 0x500)):
        f = free.clone()
        got = page_fork(lens, table, f, ring, source=source, before=_i32([before], dev))
        assert int(got.status) == want, before
        if want:
            assert got.table.tolist() == [[1, 2], [3, 0], [0, 0]] and got.lens.tolist() == [70, 3, 0] and not got.copies.any() and got.ring.tolist() == [0, 1] and torch.equal(f, free)
        else:
            assert got.table.tolist() == [[1, 2], [1, 4], [0, 0]] and got.lens.tolist() == [70, 70, 0]
    got = page_fork(lens, table, free, ring, source=_i32([7], dev), before=_i32(4, dev))  # (of any shape, as page_slots' out takes it)
    with pytest.raises(RuntimeError, match="page_fork: an impossible source.*the call before it was not done .*n_tokens"):
        got.check()
    for bad in (_i32([0, 0], dev), _i32([0], dev).long(), ring):
        with pytest.raises(ValueError):
            page_fork(lens, table, free, ring, source=source, before=bad)
    # named by the call that made the state
    pool = TokenPagePool(2, 1, 8, F16, dev)
    state = pool.step(pool.start(1, 2), _i32([70], dev), 70).check()
    with pytest.raises(RuntimeError, match="^TokenPagePool.fork: more copies needed"):
        pool.fork(state, _i32([0, 0], dev)).check()
    out = pool.fork(state, _i32([0], dev)).check()
    with pytest.raises(RuntimeError, match="^page_slots: a row would pass its table's pages"):
        page_slots(state.lens, _i32([900], dev), state.table, pool.free, pool.ring.clone(), 0, out=out).check()


# ------------------------------------------------------------------ the pool's layers and rows
def test_layers_that_do_not_fit_the_pool(dev):
    """Layers with fewer pages than the tables may name are refused ahead of the call (a move outside them is not made,
    without a word); more pages are no matter."""
    h = lambda n: torch.zeros(n, 2, 64, 16, dtype=F16, device=dev)  # noqa: E731
    pool = TokenPagePool(6, 2, 16, F16, dev)
    state = pool.step(pool.start(1, 3), _i32([100], dev), 100).check()
    path, counts = _i32([[0]], dev), _i32([1], dev)
    was = [t.clone() for t in (pool.free, pool.ring)]
    for n in (6, 3, 1):
        few = PageLayers([h(n), h(n)])
        with pytest.raises(ValueError, match="TokenPagePool.fork: layers need the pool's pages"):
            pool.fork(state, _i32([0, 0], dev), layers=few)
        with pytest.raises(ValueError, match="TokenPagePool.accept: layers need the pool's pages"):
            pool.accept(state, path, counts, few)
        with pytest.raises(ValueError, match="layers need"):
            pool.fork(state, _i32([0, 0], dev), layers=[h(n)])
    assert all(torch.equal(a, b) for a, b in zip((pool.free, pool.ring), was))
    pool.step(state, _i32([0], dev), 0, reset=torch.zeros(1, dtype=torch.bool, device=dev)).check()  # nothing was forked
    more = [h(9).normal_(), h(9)]
    state = pool.fork(state, _i32([0, 0], dev), layers=more).check()
    a, b = state.table[:, 1].tolist()
    assert a != b and torch.equal(more[0][a, :, :36], more[0][b, :, :36])


def test_clear(dev):
    """A pool that was forked takes ``reset`` again once it is cleared, with all of its pages and in the same memory."""
    pool = TokenPagePool(7, 1, 8, F16, dev)
    none = torch.zeros(2, dtype=torch.bool, device=dev)
    state = pool.step(pool.start(2, 3), _i32([130, 3], dev), 133).check()
    state = pool.fork(state, _i32([1, 0], dev)).check()
    with pytest.raises(ValueError, match="clear the pool"):
        pool.step(state, _i32([1, 1], dev), 2, reset=none)
    at = pool.free.data_ptr()
    pool.clear()
    assert pool.free.data_ptr() == at and pool.free.tolist() == [1, 2, 3, 4, 5, 6, 7] and pool.ring.tolist() == [0, 7]
    state = pool.step(pool.start(2, 3), _i32([192, 65], dev), 257).check()
    state = pool.step(state, _i32([1, 1], dev), 2, reset=torch.tensor([True, False], device=dev)).check()
    assert state.lens.tolist() == [1, 66] and state.ring.tolist()[1] == 4


# ------------------------------------------------------------------ moves of very many rows
def test_moves_of_more_workgroups_than_a_launch_has(dev):
    """Past 2^32 threads, in tensors of 16 kv heads: the copies and paths of all rows are made, the first and the last too."""
    R, Hkv, D = 2**20, 16, 8
    x = torch.randn(40, Hkv, 64, D, device=dev).half()
    layers = PageLayers([x])
    want = x.clone()
    copies = torch.zeros(R, 3, dtype=torch.int32, device=dev)
    rows = [0, 1, R // 2, R - 20, R - 17, R - 16, R - 2, R - 1]
    for i, r in enumerate(rows):
        copies[r] = _i32([1 + i, 20 + i, 5 + i], dev)
        want[20 + i, :, : 5 + i] = want[1 + i, :, : 5 + i]
    paged_copy(copies, layers)
    assert torch.equal(x, want)
    # 512 heads of 256 channels: 64 workgroups a row, 2^18 rows fill a launch
    Hkv, D, B = 512, 256, 2**18 + 5
    x = torch.randn(8, Hkv, 64, D, device=dev).half()
    layers, want = PageLayers([x]), x.clone()
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    path, counts, table, lens, starts = z(B, 2), z(B), z(B, 1), z(B), z(B + 1)
    for i, r in enumerate((0, 9, 2**18 - 2, 2**18 - 1, 2**18, B - 1)):
        path[r] = _i32([1, 3], dev)
        counts[r], table[r], lens[r] = 2, 1 + i, 10
        starts[r + 1 :] += 4  # tokens 6 .. 9 are drafted, those at 7 and 9 stay
        want[1 + i, :, 6], want[1 + i, :, 7] = want[1 + i, :, 7].clone(), want[1 + i, :, 9].clone()
    kept = paged_compact(path, counts, table, lens, starts, layers)
    assert torch.equal(x, want) and torch.equal(kept, torch.where(lens > 0, 8, 0).int())


def test_numbers_that_are_held_negated_are_refused(dev):
    """One row's number as the imaginary part of a conjugate: memory of the other sign, which looks contiguous."""
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    odd = torch.complex(torch.zeros(1, device=dev), torch.full((1,), -0.5, device=dev)).conj().imag
    assert odd.is_neg() and odd.is_contiguous() and odd.item() == 0.5
    target = torch.full((1, 4), 0.25, device=dev)
    starts = _i32([0, 1], dev)
    assert verify_drafts(target, z(1), z(1), starts, torch.zeros(1, device=dev), odd.clone().resolve_neg(), 1).next.tolist() == [2]
    for name in ("uniforms", "final"):
        with pytest.raises(ValueError, match=name):
            verify_drafts(target, z(1), z(1), starts, **{**dict(uniforms=torch.zeros(1, device=dev), final=torch.zeros(1, device=dev)), name: odd}, max_path=1)
