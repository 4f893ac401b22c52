"""Speculative steps as a program makes them: trees with filler tokens, steps that could not be done, layers that do not
fit the pool."""

from __future__ import annotations

import random

import pytest
import torch

from fade_amd.kernels import verify_drafts
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
