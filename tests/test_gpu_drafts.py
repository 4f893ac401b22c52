"""Drafted tokens on the GPU: ``draft_tree`` against the parents followed on the host, ``paged_attention`` with masks
of each token's own against a softmax in 64 bits, ``verify_drafts`` against a walk on renormalized distributions
in 64 bits and, in its results' frequencies, against the target."""

from __future__ import annotations

import math
import random

import pytest
import torch

from fade_amd import _lib
from fade_amd.kernels import PagedAttentionPlan, draft_tree, paged_attention, verify_drafts
from fade_amd.pages import PAGE_TOKENS
from test_gpu_paged import _check, _i32, _pages, _starts

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _tree(rng, n, fan=3, reach=6, chain=False):
    """Parents of a random tree of n tokens."""
    out = []
    for i in range(n):
        out.append(-1 if i == 0 else i - 1 if chain else rng.randint(max(0, i - reach), i - 1))
    return out


def _sight(parents):
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    return seen


def _words(masks, words):
    return [[(m >> 32 * w & 0xFFFFFFFF) - (m >> 32 * w + 31 & 1) * 2**32 for w in range(words)] for m in masks]


# ------------------------------------------------------------------ draft_tree
@pytest.mark.parametrize("rows", [[1], [2], [12], [0, 3, 0, 40], [64, 33, 32, 31], [1024], [1000, 1, 517], [5] * 700])
@pytest.mark.parametrize("kind", ["tree", "chain", "forest"])
def test_tree_against_the_host(dev, rows, kind):
    rng = random.Random(len(rows) + max(rows))
    trees = [_tree(rng, n, chain=kind == "chain") for n in rows]
    if kind == "forest":
        trees = [[-1 if rng.random() < 0.2 else p for p in t] for t in trees]
    lens = [n + rng.randint(0, 5000) for n in rows]
    words, pad = -(-max(rows) // 32), 5
    parents = _i32([p for t in trees for p in t] + [77] * pad, dev)
    got = draft_tree(parents, _i32(lens, dev), _i32(_starts(rows), dev), max(rows)).check()
    bits, depth, pos = [], [], []
    for L, t in zip(lens, trees):
        masks = _sight(t)
        bits += _words(masks, words)
        depth += [bin(m).count("1") - 1 for m in masks]
        pos += [L - len(t) + bin(m).count("1") - 1 for m in masks]
    assert got.bits.tolist() == bits + [[0] * words] * pad
    assert got.depth.tolist() == depth + [0] * pad and got.positions.tolist() == pos + [0] * pad
    assert got.status.tolist() == [0] * len(rows)


def test_tree_impossible_parents_and_too_many_tokens(dev):
    parents = _i32([-1, 1, 0, -7, 9, 2] + [i - 1 for i in range(40)], dev)
    got = draft_tree(parents, _i32([100, 40], dev), _i32([0, 6, 46], dev), 30)
    assert got.status.tolist() == [2, 1]
    assert got.bits[:6, 0].tolist() == [1, 2, 5, 8, 16, 37] and got.depth[:6].tolist() == [0, 0, 1, 0, 0, 2]
    assert got.bits[6:38, 0].tolist() == [(2 << i) - 1 - (2**32 if i == 31 else 0) for i in range(32)]
    assert got.bits[38:, 0].tolist() == [0] * 8 and got.depth[38:].tolist() == [0] * 8 and got.positions[38:].tolist() == [0] * 8
    with pytest.raises(RuntimeError, match="row 0: a parent"):
        got.check()
    # starts outside the tokens are kept inside them
    got = draft_tree(parents[:6], _i32([100, 40], dev), _i32([-3, 6, 99], dev), 30)
    assert got.bits[:6, 0].tolist() == [1, 2, 5, 8, 16, 37]
    assert draft_tree(parents[:0], _i32([5], dev), _i32([0, 0], dev), 1).bits.shape == (0, 1)


def test_tree_refusals(dev):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    ok = dict(parents=z(6), lens=z(2), starts=z(3), max_nodes=4)
    draft_tree(**ok)
    for bad in (dict(parents=z(6).long()), dict(parents=z(2, 3)), dict(parents=z(12)[::2]), dict(lens=z(3)), dict(starts=z(2)), dict(starts=z(3).float()),
                dict(max_nodes=0), dict(max_nodes=1025)):
        with pytest.raises(ValueError):
            draft_tree(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        draft_tree(**{**ok, "lens": z(2).cpu()})


# ------------------------------------------------------------------ attention
def _reference(q, k_pages, v_pages, table, lens, starts, scale, masks):
    """(output, tolerance) in 64 bits: a rounding of the output, of each probability and of the scores' fp32 sums.
    masks[t]: the row's new tokens that token t sees, as a number's bits."""
    T, Hq, D = q.shape
    Hkv = k_pages.shape[1]
    G, u = Hq // Hkv, torch.finfo(q.dtype).eps / 2
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b, L in enumerate(lens):
        s, e = starts[b], starts[b + 1]
        n = e - s
        if n == 0 or L == 0:
            continue
        ids = table[b, : -(-L // PAGE_TOKENS)].long()
        seen = torch.tensor([[j < L - n or bool(masks[t] >> (j - (L - n)) & 1) for j in range(L)] for t in range(s, e)], device=q.device)
        for h in range(Hkv):
            k, v = (x[ids, h].double().reshape(-1, D)[:L] for x in (k_pages, v_pages))
            qh = q[s:e, h * G : (h + 1) * G].double().transpose(0, 1).reshape(G * n, D)
            vis = seen.repeat(G, 1)
            x = (qh @ k.t()) * scale
            p = torch.softmax(x.masked_fill(~vis, -math.inf), dim=-1).nan_to_num(0.0)
            o = p @ v
            # a score's fp32 sum: D products, each addition 2^-24 of the sum of their sizes, and a few more; the
            # maximum's own error cancels
            ds = ((D + 8) * 2.0**-24 * scale * (qh.abs() @ k.abs().t())).masked_fill(~vis, 0.0).amax(-1, keepdim=True)
            # fp16 probabilities under 2^-14 of the maximum's lose up to 2^-25 each, absolutely
            small = 2.0**-25 * vis.sum(-1, keepdim=True) * v.abs().amax() * p.amax(-1, keepdim=True) if q.dtype == F16 else 0.0
            t = u * o.abs() + (2 * u + 2 * ds) * (1 + u) * (p @ v.abs()) + small + torch.finfo(q.dtype).tiny
            out[s:e, h * G : (h + 1) * G] = o.reshape(G, n, D).transpose(0, 1)
            tol[s:e, h * G : (h + 1) * G] = t.reshape(G, n, D).transpose(0, 1)
    return out, tol


# a row's tokens (the drafted ones included), its drafted ones
ROWS = {
    "one": ([1], [1]),
    "few": ([70, 5, 1300], [4, 5, 3]),
    "chat": ([1008], [8]),
    "ragged": ([64, 500, 129, 33, 1000], [17, 37, 64, 33, 25]),
    "no_prefix": ([9, 70, 130], [9, 70, 130]),
    "page_ends": ([64 + 32, 128, 192 - 1, 65, 640], [32, 64, 63, 1, 96]),
    "empty": ([0, 40, 10, 0, 200], [0, 0, 4, 0, 3]),
    "mixed": ([2000, 900, 31, 65], [1, 333, 31, 1]),
    "many": ([(37 * i) % 150 + 3 for i in range(70)], [i % 4 for i in range(70)]),
}


def _masks(rng, kind, rows):
    out = []
    for n in rows:
        if kind == "tree":
            out += _sight(_tree(rng, n))
        else:  # any tokens, none too
            out += [rng.getrandbits(n) if rng.random() < 0.8 else 0 for _ in range(n)]
    return out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", list(ROWS))
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (14, 2, 64), (16, 8, 256), (3, 3, 128), (20, 1, 64), (6, 2, 80), (4, 4, 8), (2, 1, 200)])
def test_tree_attention(dev, Hq, Hkv, D, rows, dtype):
    lens, new = ROWS[rows]
    rng = random.Random(D + len(rows))
    g = torch.Generator(device=dev).manual_seed(D + len(rows))
    k, v, table = _pages(g, dev, lens, Hkv, D, dtype, junk=math.nan)  # what stands where no token does must not count
    q = torch.randn(sum(new), Hq, D, generator=g, device=dev).to(dtype)
    starts = _starts(new)
    for kind in ("tree", "any"):
        masks = _masks(rng, kind, new)
        words = -(-max(new) // 32)
        want, tol = _reference(q, k, v, table, lens, starts, 1 / math.sqrt(D), masks)
        # bits past a row's tokens say nothing
        tree = _i32(_words([m | (-1 << n) & (1 << 32 * words) - 1 for m, n in zip(masks, [n for n in new for _ in range(n)])], words), dev).view(-1, words)
        args = (q, k, v, table, _i32(lens, dev), _i32(starts, dev))
        got = paged_attention(*args, mask="tree", tree=tree)
        _check(got, want, tol, kind)
        assert torch.equal(got, paged_attention(*args, mask="tree", tree=torch.nn.functional.pad(tree, (0, 3), value=-1)))
        # words that are not there: their tokens are not seen
        if words > 1:
            short = [m & 0xFFFFFFFF for m in masks]
            want, tol = _reference(q, k, v, table, lens, starts, 1 / math.sqrt(D), short)
            _check(paged_attention(*args, mask="tree", tree=tree[:, :1].contiguous()), want, tol, "one word")


@pytest.mark.parametrize("D", [64, 128, 256])
def test_chains_are_the_causal_mask(dev, D):
    """A chain's masks, as ``draft_tree`` gives them, are the bottom-right causal mask."""
    lens, new = [300, 77, 1000, 64], [3, 77, 130, 2]
    g = torch.Generator(device=dev).manual_seed(3)
    k, v, table = _pages(g, dev, lens, 2, D, BF16)
    q = torch.randn(sum(new), 8, D, generator=g, device=dev).bfloat16()
    args = (q, k, v, table, _i32(lens, dev), _i32(_starts(new), dev))
    tree = draft_tree(_i32([i - 1 for n in new for i in range(n)], dev), args[4], args[5], max(new)).check()
    want, tol = _reference(q, k, v, table, lens, _starts(new), 1 / math.sqrt(D), [(2 << i) - 1 for n in new for i in range(n)])
    _check(paged_attention(*args, mask="tree", tree=tree.bits), want, tol, "tree")
    _check(paged_attention(*args), want, tol, "causal")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (3, 3, 64), (4, 2, 256), (2, 1, 80)])
@pytest.mark.parametrize("lens,new", [([70, 33, 200], [3, 4, 2]), ([64, 300], [64, 170]), ([130, 1, 700], [130, 1, 97])])
def test_tree_attention_values_that_are_no_numbers(dev, lens, new, Hq, Hkv, D, dtype):
    """An infinity or a NaN in V reaches the queries that see its key, and no other."""
    rng = random.Random(D)
    g = torch.Generator(device=dev).manual_seed(D)
    k, v, table = _pages(g, dev, lens, Hkv, D, dtype, junk=math.nan)
    q = torch.randn(sum(new), Hq, D, generator=g, device=dev).to(dtype)
    starts, masks, words = _starts(new), [], -(-max(new) // 32)
    for n in new:
        masks += _sight(_tree(rng, n))
    args = (table, _i32(lens, dev), _i32(starts, dev))
    tree = dict(mask="tree", tree=_i32(_words(masks, words), dev))
    odd = v.clone()
    up, down = torch.zeros(2, len(lens), max(lens), Hkv, D, dtype=torch.bool, device=dev)
    for b, (L, n) in enumerate(zip(lens, new)):
        for j, (t, x) in enumerate(zip((L - 1, L - 1 - n // 2, max(L - n - 1, 0)), (math.nan, math.inf, -math.inf))):
            at = (table[b, t // PAGE_TOKENS], (b + j) % Hkv, t % PAGE_TOKENS)
            odd[(*at, slice(j, D, 5))] = x
            v[(*at, slice(j, D, 5))] = 0.0
            up[b, t, (b + j) % Hkv, j::5] |= not x < 0
            down[b, t, (b + j) % Hkv, j::5] |= not x > 0
    want, got = paged_attention(q, k, v, *args, **tree), paged_attention(q, k, odd, *args, **tree)
    for b, (L, n) in enumerate(zip(lens, new)):
        for i in range(n):
            seen = torch.tensor([j < L - n or bool(masks[starts[b] + i] >> (j - (L - n)) & 1) for j in range(L)], device=dev)
            for kind, sign in ((up, math.inf), (down, -math.inf)):
                hit = (kind[b, :L] & seen[:, None, None]).any(0).repeat_interleave(Hq // Hkv, 0)
                want[starts[b] + i] = torch.where(hit, want[starts[b] + i] + sign, want[starts[b] + i])
    wrong = ~((got == want) | (got.isnan() & want.isnan()))
    at = wrong.nonzero()[:4].tolist()
    assert not at, [(i, float(got[tuple(i)]), float(want[tuple(i)])) for i in at]


@pytest.mark.parametrize("new", [1, 3, 40])
def test_tree_attention_strides_tail_and_scale(dev, new):
    g = torch.Generator(device=dev).manual_seed(new)
    rng = random.Random(new)
    lens, Hq, Hkv, D = [500, 1200, 64], 12, 4, 128
    starts = _starts([new] * 3)
    k, v, table = _pages(g, dev, lens, Hkv, D, F16)
    T = starts[-1] + 9
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=dev).half()
    q = qkv[:, :Hq]
    masks = _masks(rng, "tree", [new] * 3)
    tree = _i32(_words(masks + [-1 & 2**64 - 1] * 9, 2), dev)
    args, kw = (q, k, v, table, _i32(lens, dev), _i32(starts, dev)), dict(mask="tree", tree=tree, sm_scale=0.3)
    want, tol = _reference(q, k, v, table, lens, starts, 0.3, masks)
    got = paged_attention(*args, **kw)
    _check(got, want, tol)
    assert not got[starts[-1] :].any()  # a new tensor: zeros behind the last sequence
    out = torch.full((Hq, T, D + 8), 7.0, device=dev).half()[:, :, 4 : 4 + D].transpose(0, 1)
    assert paged_attention(*args, **kw, out=out) is out and torch.equal(out[: starts[-1]], got[: starts[-1]])
    assert bool((out[starts[-1] :] == 7.0).all())  # the caller's: left as they were
    mine = q.clone()
    assert torch.equal(paged_attention(mine, *args[1:], **kw, out=mine)[: starts[-1]], got[: starts[-1]])


def test_tree_attention_device_data_out_of_range(dev):
    """Fewer tokens than new ones, lengths and starts that cannot be: kept inside the tensors."""
    H, D = 2, 64
    g = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.randn(4, H, PAGE_TOKENS, D, generator=g, device=dev).half() for _ in range(2))
    q = torch.randn(40, H, D, generator=g, device=dev).half()
    tree = torch.full((40, 2), -1, dtype=torch.int32, device=dev)
    table = _i32([[1, 2], [3, 99]], dev)
    for lens, starts in (([20, 64], [0, 30, 40]), ([-3, 2**31 - 1], [0, 30, 2**31 - 1]), ([128, 128], [-9, 39, 7])):
        got = paged_attention(q, k, v, table, _i32(lens, dev), _i32(starts, dev), mask="tree", tree=tree)
        assert not bool(got.isnan().any())
    # 20 tokens with 30 new ones: the last new token is token 19, so the first 10 have no place; all see all 20 keys
    got = paged_attention(q, k, v, table, _i32([20, 0], dev), _i32([0, 30, 30], dev), mask="tree", tree=tree)
    want = paged_attention(q, k, v, table, _i32([20, 0], dev), _i32([0, 30, 30], dev), mask="none")
    assert bool(((got - want).abs() <= 2.0**-8).all())


def test_tree_attention_refusals(dev):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    h = lambda *s: torch.zeros(s, dtype=F16, device=dev)  # noqa: E731
    ok = dict(q=h(3, 4, 64), k_pages=h(5, 2, 64, 64), v_pages=h(5, 2, 64, 64), table=z(2, 3), lens=z(2), starts=z(3), mask="tree", tree=z(3, 1))
    paged_attention(**ok)
    buf = torch.zeros(3 * 4 * 64 + 8, dtype=F16, device=dev)
    for bad in (dict(tree=None), dict(mask="none"), dict(mask="bottom_right"), dict(tree=z(4, 1)), dict(tree=z(3)), dict(tree=z(3, 0)), dict(tree=z(3, 1).long()),
                dict(tree=z(3, 2)[:, :1]), dict(out=buf[8:].view(3, 4, 64), tree=buf[2:8].view(torch.int32).view(3, 1)),
                dict(out=buf[:-8].view(3, 4, 64), tree=buf[8:14].view(torch.int32).view(3, 1))):
        if "out" in bad and bad["tree"].data_ptr() < bad["out"].data_ptr():
            paged_attention(**{**ok, **bad})  # (beside one another)
            continue
        with pytest.raises(ValueError):
            paged_attention(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_attention(**{**ok, "tree": ok["tree"].cpu()})
    assert paged_attention(**{**ok, "q": h(0, 4, 64), "tree": z(0, 1)}).shape == (0, 4, 64)


def test_tree_attention_plans_streams_graph(dev):
    g = torch.Generator(device=dev).manual_seed(5)
    lens, new, H, D = [3000, 200, 1500], [20, 3, 64], 4, 128
    k, v, table = _pages(g, dev, lens, H, D, F16)
    lt, st = _i32(lens, dev), _i32(_starts(new), dev)
    q = torch.randn(sum(new), 4 * H, D, generator=g, device=dev).half()
    rng = random.Random(1)
    trees = [_i32(_words([m for n in new for m in _sight(_tree(rng, n))], 2), dev) for _ in range(4)]
    tree = trees[0].clone()
    plan = PagedAttentionPlan(q, k, v, table, lt, st, mask="tree", tree=tree)
    plan.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
    side = torch.cuda.Stream(dev)
    for t in trees:
        tree.copy_(t)
        plan.out.zero_()
        graph.replay()
        got = plan.out.clone()
        want = paged_attention(q, k, v, table, lt, st, mask="tree", tree=t)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = paged_attention(q, k, v, table, lt, st, mask="tree", tree=t)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(other, want)


# ------------------------------------------------------------------ verify_drafts
def _walk(target, draft, tokens, parents, uniforms, final, max_path):
    """One row, in 64 bits on the host: (path, next).  Distributions are renormalized after each refusal."""
    clean = lambda x: torch.where(x > 0, x, 0.0).double()  # noqa: E731
    V, n = target.shape[1], len(parents)
    if n == 0:
        return [], -1
    node, path = 0, [0]
    while True:
        p = clean(target[node])
        first = p.clone()
        q = None if draft is None else clean(draft[node])
        go, kids, stock = None, [i for i in range(1, n) if parents[i] == node] if len(path) < max_path else [], 1.0
        for c in kids:
            x, u = tokens[c], uniforms[c]
            px = float(p[x]) if 0 <= x < V else 0.0
            qx = 0.0 if q is None or not 0 <= x < V else float(q[x])
            if px > 0 and (u * stock < px if q is None else u * qx * stock < px):
                go = c
                break
            if q is None:
                stock -= px
                if 0 <= x < V:
                    p[x] = 0.0
            else:
                p = (p - q * stock).clamp(min=0)
                stock = float(p.sum())
        if go is None:
            break
        node = go
        path.append(go)
    if not float(p.sum()) > 0:
        p = first
    if not float(p.sum()) > 0:
        return path, -1
    c = p.cumsum(0)
    past = ((c > final * float(c[-1])) & (p > 0)).nonzero()
    return path, int(past[0]) if past.numel() else int(p.nonzero()[-1])


def _verified(dev, target, draft, tokens, trees, uniforms, final, max_path, tok=torch.int64):
    starts = _starts([len(t) for t in trees])
    parents = _i32([p for t in trees for p in t], dev)
    got = verify_drafts(target, torch.tensor(tokens, dtype=tok, device=dev), parents, _i32(starts, dev), torch.tensor(uniforms, dtype=F32, device=dev),
                        torch.tensor(final, dtype=F32, device=dev), max_path, draft=draft)
    assert got.tokens.dtype == got.next.dtype == tok
    uniforms, final = torch.tensor(uniforms, dtype=F32).tolist(), torch.tensor(final, dtype=F32).tolist()
    t, d = target.cpu(), None if draft is None else draft.cpu()
    path, counts, tokens_out, nxt = [], [], [], []
    for b, tree in enumerate(trees):
        s, e = starts[b], starts[b + 1]
        p, x = _walk(t[s:e], None if d is None else d[s:e], tokens[s:e], tree, uniforms[s:e], final[b], max_path)
        path.append(p + [-1] * (max_path - len(p)))
        counts.append(len(p))
        out = [tokens[s + i] for i in p[1:]] + ([x] if p else [])
        tokens_out.append(out + [-1] * (max_path - len(out)))
        nxt.append(x)
    assert got.path.tolist() == path
    assert got.counts.tolist() == counts and got.tokens.tolist() == tokens_out and got.next.tolist() == nxt
    return got


def _probs(g, dev, T, V, dtype, peak=3.0):
    z = peak * torch.randn(T, V, generator=g, device=dev)
    near = z + 0.8 * torch.randn(T, V, generator=g, device=dev)
    return torch.softmax(z, -1).to(dtype), torch.softmax(near, -1).to(dtype)


def _drafted(rng, draft, trees, dup=0.1):
    """Tokens from each parent's probabilities, some of them a sibling's once more."""
    out, at, d = [], 0, draft.float().cpu()
    for tree in trees:
        row = []
        for i, p in enumerate(tree):
            same = [row[j] for j in range(1, i) if tree[j] == p]
            if same and rng.random() < dup:
                row.append(rng.choice(same))
                continue
            row.append(int(torch.multinomial(d[at + max(p, 0)].clamp(min=0) + 1e-30, 1)))
        out += row
        at += len(tree)
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("V,rows", [(1, [3, 1]), (2, [4, 2, 0, 5]), (7, [12] * 9), (63, [1, 2, 30]), (300, [70, 9, 0, 1]), (1001, [17] * 5), (4097, [9, 64, 65, 130]),
                                    (32000, [6, 5]), (151936, [12, 3]), (20000, [1024, 2])])
def test_verify_against_the_host(dev, V, rows, with_draft, dtype):
    torch.manual_seed(V)
    rng = random.Random(V + len(rows))
    g = torch.Generator(device=dev).manual_seed(V)
    trees = [_tree(rng, n, reach=5) for n in rows]
    target, draft = _probs(g, dev, sum(rows), V, dtype)
    tokens = _drafted(rng, draft, trees)
    for k in range(3):
        u = [rng.random() * (0.3 if k == 1 else 1) for _ in tokens]
        f = [rng.random() for _ in rows]
        _verified(dev, target, draft if with_draft else None, tokens, trees, u, f, max(rows) if k < 2 else 3, torch.int64 if k else torch.int32)


@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_strides_and_alignment(dev, with_draft):
    g = torch.Generator(device=dev).manual_seed(2)
    rng = random.Random(2)
    trees = [_tree(rng, n) for n in (9, 6)]
    V = 1003
    for dtype, lead, width in ((F32, 1, 1007), (F32, 3, 1006), (BF16, 1, 1005), (F16, 7, 1013)):
        bufs = [torch.zeros(15, width, dtype=dtype, device=dev) for _ in range(2)]
        target, draft = (b[:, lead : lead + V] for b in bufs)
        t, d = _probs(g, dev, 15, V, dtype)
        target.copy_(t)
        draft.copy_(d)
        for b in bufs:  # what lies beside the rows must not count
            b[:, :lead] = 1e4
            b[:, lead + V :] = 1e4
        tokens = _drafted(rng, draft, trees)
        u, f = [rng.random() for _ in tokens], [rng.random(), rng.random()]
        _verified(dev, target, draft if with_draft else None, tokens, trees, u, f, 9)
        # draft of another alignment than target's, and one row for all tokens
        _verified(dev, target, d if with_draft else None, tokens, trees, u, f, 9)
        _verified(dev, t[:1].expand(15, V), d[3:4].expand(15, V) if with_draft else None, tokens, trees, u, f, 9)


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_verify_borders(dev, with_draft, dtype):
    """Uniform numbers of 0 and almost 1, equal distributions, one-hot ones, tokens outside the vocabulary, NaN."""
    V, tree = 130, [-1, 0, 0, 0, 1, 4, 4]
    eps = torch.finfo(F32).eps
    g = torch.Generator(device=dev).manual_seed(9)
    target, draft = _probs(g, dev, 7, V, dtype)
    args = (dev, target)
    d = draft if with_draft else None
    for u in (0.0, 1.0 - eps / 2):
        for f in (0.0, 1.0 - eps / 2, 0.5):
            _verified(dev, target, d, [5, 17, 17, 90, 129, 0, 3], [tree], [u] * 7, [f], 7)
    # equal distributions: always accepted while drawn from them, nothing left after a refusal of chance
    _verified(dev, target, target.clone() if with_draft else None, [5, 17, 3, 90, 129, 0, 3], [tree], [0.999] * 7, [0.7], 7)
    # a one-hot target: its token is accepted, any other refused
    hot = torch.zeros_like(target)
    hot[torch.arange(7), torch.tensor([3, 64, 64, 1, 129, 0, 2])] = 1.0
    got = _verified(dev, hot, d, [0, 7, 3, 3, 64, 129, 129], [tree], [0.5] * 7, [0.999], 7)
    assert got.path[0, :2].tolist() == [0, 2] and got.next.tolist() == [64]
    got = _verified(dev, hot, hot.clone() if with_draft else None, [0, 3, 3, 3, 64, 129, 129], [tree], [0.5] * 7, [0.0], 7)
    assert got.path[0].tolist() == [0, 1, 4, 5, -1, -1, -1] and got.next.tolist() == [0]
    # tokens outside the vocabulary are refused
    _verified(dev, target, d, [0, -1, V, 2**31 - 1, 3, 4, 5], [tree], [0.0] * 7, [0.3], 7)
    # NaN and negative entries have no weight; a target without any gives no token
    odd = target.clone()
    odd[:, ::3] = math.nan
    odd[:, 1::3] *= -1
    _verified(dev, odd, d, [0, 2, 3, 5, 8, 11, 4], [tree], [0.5] * 7, [0.4], 7)
    none = torch.full_like(target, math.nan)
    got = _verified(dev, none, d, [0, 2, 3, 5, 8, 11, 4], [tree], [0.5] * 7, [0.4], 7)
    assert got.next.tolist() == [-1] and got.tokens[0, 0] == -1 and got.counts.tolist() == [1]
    # tokens that follow none, or a later one, are never reached
    got = verify_drafts(target, _i32([0, 3, 4, 5, 6, 7, 8], dev), _i32([-1, -1, 2, 9, -5, 5, 6], dev), _i32([0, 7], dev), torch.zeros(7, device=dev),
                        torch.zeros(1, device=dev), 7, draft=d)
    assert got.counts.tolist() == [1]


@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_keeps_the_targets_distribution(dev, with_draft):
    """The first token that comes out is distributed as the target says, whatever was drafted."""
    V, B, n = 6, 60000, 4
    g = torch.Generator(device=dev).manual_seed(4)
    p = torch.tensor([0.35, 0.05, 0.25, 0.02, 0.3, 0.03], device=dev)
    q = torch.tensor([0.1, 0.4, 0.2, 0.05, 0.05, 0.2], device=dev)
    parents = _i32([-1, 0, 0, 0] * B, dev)
    starts = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=dev)
    if with_draft:
        tokens = torch.multinomial(q, B * n, replacement=True, generator=g)
    else:
        tokens = torch.tensor([0, 1, 4, 3], device=dev).repeat(B)
    got = verify_drafts(p.expand(B * n, V), tokens, parents, starts, torch.rand(B * n, generator=g, device=dev), torch.rand(B, generator=g, device=dev), 2,
                        draft=q.expand(B * n, V) if with_draft else None)
    share = torch.bincount(got.tokens[:, 0], minlength=V).double() / B
    # six deviations of a share of B drawings
    assert bool(((share - p.double()).abs() <= 6 * (p * (1 - p) / B).sqrt().double()).all()), share.tolist()
    assert 0.2 < float((got.counts == 2).double().mean()) < 0.99


@pytest.mark.parametrize("wait", [True, False])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("rows,V", [([15], 70000), ([15, 3, 0, 9], 50000), ([12] * 40, 40011), ([12] * 3, 9000)])
def test_verify_many_refusals(dev, monkeypatch, rows, V, with_draft, wait):
    """Stars, whose children are all refused or nearly so: more sums than a row's workgroups share, with and without
    their wait for one another."""
    if not wait:
        launch = _lib.launch_with_workspace

        def without(name, args, device):
            args.polls = -1
            launch(name, args, device)

        monkeypatch.setattr(_lib, "launch_with_workspace", without)
    rng = random.Random(V)
    torch.manual_seed(V)
    g = torch.Generator(device=dev).manual_seed(V)
    trees = [[-1] + [0] * (n - 1) if n else [] for n in rows]
    target, draft = _probs(g, dev, sum(rows), V, F32, peak=1.0)
    tokens = _drafted(rng, draft, trees, dup=0.2)
    for u in (0.9999, 0.97):
        _verified(dev, target, draft if with_draft else None, tokens, trees, [u] * len(tokens), [rng.random() for _ in rows], 4)
    # nothing left after the refusals: drawn from the target itself
    same = target[:1].expand(sum(rows), V)
    _verified(dev, same, same if with_draft else None, tokens, trees, [0.9999] * len(tokens), [rng.random() for _ in rows], 4)


def test_verify_rows_far_apart(dev):
    """Rows whose offsets pass 2^32 elements."""
    V, st = 1000, 2**31 + 64
    g = torch.Generator(device=dev).manual_seed(6)
    t, d = _probs(g, dev, 4, V, BF16)
    spare = torch.empty(3 * st + V, dtype=BF16, device=dev)
    far = spare.as_strided((4, V), (st, 1))
    far.copy_(t)
    tokens = _drafted(random.Random(1), d, [[-1, 0, 1, 2]])
    for u in (0.0, 0.9):
        _verified(dev, far, d, tokens, [[-1, 0, 1, 2]], [u] * 4, [0.6], 4)
        _verified(dev, d, far, tokens, [[-1, 0, 1, 2]], [u] * 4, [0.6], 4)


@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_more_rows_than_workgroups_at_once(dev, with_draft):
    """Rows so many that each has one workgroup, whatever the vocabulary."""
    rng = random.Random(11)
    g = torch.Generator(device=dev).manual_seed(11)
    trees = [[-1, 0, 0][: rng.randint(1, 3)] for _ in range(300)]
    T = sum(map(len, trees))
    target, draft = _probs(g, dev, T, 40960, BF16)
    tokens = _drafted(rng, draft, trees)
    _verified(dev, target, draft if with_draft else None, tokens, trees, [rng.random() for _ in tokens], [rng.random() for _ in trees], 3)


def test_verify_graph_streams_and_repeats(dev):
    g = torch.Generator(device=dev).manual_seed(8)
    rng = random.Random(8)
    trees = [_tree(rng, n, reach=3) for n in (12, 9, 0, 5)]
    T, V = 26, 40000
    sets = []
    for _ in range(4):
        target, draft = _probs(g, dev, T, V, F32)
        sets.append((target, torch.tensor(_drafted(rng, draft, trees), device=dev), torch.rand(T, generator=g, device=dev), torch.rand(4, generator=g, device=dev), draft))
    parents, starts = _i32([p for t in trees for p in t], dev), _i32(_starts([len(t) for t in trees]), dev)
    call = lambda x: verify_drafts(x[0], x[1], parents, starts, x[2], x[3], 12, draft=x[4])  # noqa: E731
    want = [call(x) for x in sets]
    bufs = tuple(t.clone() for t in sets[0])
    call(bufs)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(call(bufs))
    side = torch.cuda.Stream(dev)
    same = lambda a, b: all(torch.equal(getattr(a, f), getattr(b, f)) for f in ("path", "counts", "tokens", "next"))  # noqa: E731
    for i in range(8):
        for dst, src in zip(bufs, sets[i % 4]):
            dst.copy_(src)
        for t in (outs[i % 2].path, outs[i % 2].counts, outs[i % 2].tokens, outs[i % 2].next):
            t.fill_(-9)
        graphs[i % 2].replay()
        assert same(outs[i % 2], want[i % 4]), i
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            a = call(sets[i % 4])
        b = call(sets[(i + 1) % 4])
        torch.cuda.synchronize()
        assert same(a, want[i % 4]) and same(b, want[(i + 1) % 4])


def test_verify_refusals(dev):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    f = lambda *s: torch.zeros(s, device=dev)  # noqa: E731
    ok = dict(target=f(6, 50), tokens=z(6), parents=z(6), starts=z(3), uniforms=f(6), final=f(2), max_path=4, draft=f(6, 50))
    verify_drafts(**ok)
    for bad in (dict(target=f(6, 50).double()), dict(target=f(6, 50).long()), dict(target=f(300)), dict(target=f(50, 6).t()), dict(target=f(5, 50)), dict(draft=f(6, 49)),
                dict(draft=f(6, 50).half()), dict(draft=f(50, 6).t()), dict(tokens=z(5)), dict(tokens=z(6).short()), dict(tokens=z(2, 3)), dict(parents=z(6).long()),
                dict(starts=z(4)), dict(uniforms=f(6).double()), dict(uniforms=f(7)), dict(final=f(2).half()), dict(final=f(2, 1)), dict(max_path=0),
                dict(max_path=1025), dict(target=f(6, 0), draft=f(6, 0)), dict(target=f(6, 50).requires_grad_()), dict(draft=f(6, 50).requires_grad_()),
                dict(uniforms=f(6).requires_grad_())):
        with pytest.raises(ValueError):
            verify_drafts(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        verify_drafts(**{**ok, "final": ok["final"].cpu()})
    assert verify_drafts(f(0, 50), z(0), z(0), z(2), f(0), f(1), 3).next.tolist() == [-1]
