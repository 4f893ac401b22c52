"""Operators of speculative decoding and of branching rows over the paged 16-bit KV cache that are timed.

Five kinds of work, each through the entry points that a serving program calls:

  tree     ``draft_tree``: from every drafted token's parent, its depth, its rotary
           position and the bits of the tokens that it sees
  attend   ``PagedAttentionPlan`` with the mask "tree": the drafted tokens of every row
           over the row's pages, each seeing the row's tokens and its own ancestors
  verify   ``verify_drafts``: the path of drafted tokens that the target's probabilities
           accept, and the token behind it
  accept   ``paged_compact`` and ``page_fork``: the accepted tokens' K and V to
           consecutive places in every layer, the pages behind them returned
  fork     ``page_fork`` and ``paged_copy``: rows that go on from other rows (samples of
           one prompt, beams), sharing full pages, with a copy of the page that each
           goes on writing; dropped and shortened rows' pages returned

Inputs follow the benchmark's distributions: K ~ N(0, 1) with per-channel scales
~ LogNormal(0, 0.5), V and Q ~ N(0, 1).  With ``own`` false every operator is
computed in its plain form.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
PAGE = 64
WHOLE = 2**31 - 1
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# query heads, kv heads, head_dim: 8B-class GQA-4, Qwen2.5-7B's GQA-7, a 70B-class
# GQA-8, Qwen2.5-0.5B's 14/2 at head_dim 64, Gemma's 16/8 at head_dim 256
SHAPES = ((32, 8, 128), (28, 4, 128), (64, 8, 128), (14, 2, 64), (16, 8, 256))
# bounds of one case's size: elements of the K pages, attention's operations, the plain form's padded
# scores, target probabilities, elements of all layers' pages
MOST_PAGED = 16 * 8 * 8192 * 128
MOST_FLOPS = 1.8e11
MOST_SCORES = 2.6e9
MOST_PROBS = 5.5e7
MOST_LAYERS = 8.0e8


# ------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one chat's drafted tokens: a call of a few numbers, latency only
        dict(name="tree_b1", kind="tree", B=1, nodes=12, fan=3),
        # a large server's step, 64 drafted tokens a row
        dict(name="tree_b256", kind="tree", B=256, nodes=64, fan=4),
        # a small model checks eight drafted tokens of one chat
        dict(name="attend_b1_d64", kind="attend", B=1, Hq=14, Hkv=2, D=64, Lmin=1000, Lmax=1000, nodes=8, fan=2, dtype="fp16"),
        # the headline workload's layer before its compression, 16 drafted tokens a row
        dict(name="attend_b16_8k", kind="attend", B=16, Hq=32, Hkv=8, D=128, Lmin=8192, Lmax=8192, nodes=16, fan=3, dtype="fp16"),
        # a server's step: rows from short to very long, up to 48 drafted tokens, 7 query heads per kv head
        dict(name="attend_ragged_bf16", kind="attend", B=61, Hq=28, Hkv=4, D=128, Lmin=190, Lmax=32000, nodes=48, fan=4, dtype="bf16"),
        # a chain of five drafted tokens of one chat, a small vocabulary
        dict(name="verify_b1_chain", kind="verify", B=1, nodes=6, fan=1, V=32000, draft=True, dtype="fp32"),
        # a server's step: trees drawn from a draft model, a vocabulary of 152064
        dict(name="verify_b32_tree", kind="verify", B=32, nodes=12, fan=3, V=152064, draft=True, dtype="fp32"),
        # drafts without probabilities (the likeliest tokens, or found in the prompt), 16-bit probabilities
        dict(name="verify_b48_points", kind="verify", B=48, nodes=25, fan=4, V=128256, draft=False, dtype="bf16"),
        # one chat's accepted tokens in the 24 layers of a small model
        dict(name="accept_b1", kind="accept", B=1, nodes=8, fan=2, held=1000, layers=24, Hkv=2, D=64, dtype="fp16"),
        # a server's step in 28 layers
        dict(name="accept_b64", kind="accept", B=64, nodes=24, fan=3, held=500, layers=28, Hkv=4, D=128, dtype="bf16"),
        # one prompt goes on as four samples
        dict(name="fork_samples", kind="fork", groups=1, beams=1, out=4, held=1000, drops=0, cuts=0, layers=24, Hkv=2, D=64, dtype="fp16"),
        # a beam search's step in 16 layers: 24 searches of four beams, some rows dropped, some shortened
        dict(name="fork_beams", kind="fork", groups=24, beams=4, out=4, held=1100, drops=7, cuts=5, layers=16, Hkv=8, D=128, dtype="bf16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng) -> dict:
    kind = rng.choice(("tree", "attend", "attend", "attend", "verify", "verify", "accept", "fork"))
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "tree":
        nodes = _log_int(rng, 1, 256)
        return dict(kind=kind, B=_log_int(rng, 1, max(1, min(512, 16384 // nodes))), nodes=nodes, fan=rng.randint(1, 6))
    if kind == "verify":
        V, nodes = _log_int(rng, 1000, 200000), _log_int(rng, 1, 64)
        return dict(kind=kind, B=_log_int(rng, 1, max(1, min(128, int(MOST_PROBS / (V * nodes))))), nodes=nodes, fan=rng.randint(1, 4), V=V,
                    draft=rng.random() < 0.6, dtype=rng.choice(("fp32", "fp32", dtype)))
    Hq, Hkv, D = rng.choice(SHAPES[:1] * 2 + SHAPES)
    if kind == "attend":
        B, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 100)
        most = min(MOST_FLOPS / (4.0 * Hq * D), MOST_SCORES / Hq) / (B * nodes)
        Lmax = _log_int(rng, 16, max(16, int(min(32000, MOST_PAGED // (B * Hkv * D), most))))
        return dict(kind=kind, B=B, Hq=Hq, Hkv=Hkv, D=D, Lmin=max(1, Lmax // rng.choice((1, 4, 100))), Lmax=Lmax, nodes=nodes,
                    fan=rng.randint(1, 5), dtype=dtype)
    layers, held = _log_int(rng, 1, 28), _log_int(rng, 16, 4000)
    rows = int(MOST_LAYERS / (2 * layers * Hkv * D * (held + 400)))
    if kind == "accept":
        return dict(kind=kind, B=_log_int(rng, 1, max(1, min(64, rows))), nodes=_log_int(rng, 1, 64), fan=rng.randint(1, 4), held=held,
                    layers=layers, Hkv=Hkv, D=D, dtype=dtype)
    beams, out = rng.randint(1, 6), rng.randint(1, 6)
    groups = _log_int(rng, 1, max(1, min(24, rows // 6)))
    return dict(kind=kind, groups=groups, beams=beams, out=out, held=held, drops=rng.randint(0, groups * out // 4),
                cuts=rng.randint(0, groups * out // 4), layers=layers, Hkv=Hkv, D=D, dtype=dtype)


# ----------------------------------------------------------------- the inputs
def _log_lengths(rng, n: int, lo: int, hi: int) -> list[int]:
    """n lengths spread evenly over the logarithm of lo..hi, in an order of the seed's."""
    if n == 1:
        return [hi]
    out = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    rng.shuffle(out)
    return out


def _spread(rng, n: int, lo: int, hi: int) -> list[int]:
    """n numbers spread evenly over lo..hi, in an order of the seed's (one alone: hi)."""
    out = [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]
    rng.shuffle(out)
    return out


def _starts(new: list[int]) -> list[int]:
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _i32(x) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _trees(case: dict, seed: int) -> list[list[int]]:
    """Every row's drafted tokens as their parents: the first one (-1) is the row's last known token, each other
    one hangs on one of the tokens before it, at most ``fan`` on one.  Half of ``nodes`` to all of them in a row."""
    rng = random.Random(seed)
    rows = []
    for n in _spread(rng, case["B"], (case["nodes"] + 1) // 2, case["nodes"]):
        parents, kids, reach = [-1], [0] * n, max(1, n // 3)
        for i in range(1, n):
            free = [j for j in range(max(0, i - reach), i) if kids[j] < case["fan"]] or [i - 1]
            parents.append(rng.choice(free))
            kids[parents[-1]] += 1
        rows.append(parents)
    return rows


def _flat(rows: list[list[int]], pad: int = 0) -> torch.Tensor:
    return _i32([p for row in rows for p in row] + [0] * pad)


def _sight(rows: list[list[int]], words: int) -> torch.Tensor:
    """The bits of the tokens that each drafted token sees (its ancestors and itself), int32 [tokens, words]."""
    out = []
    for parents in rows:
        seen = []
        for i, p in enumerate(parents):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        out += [[(m >> 32 * w & 0xFFFFFFFF) - (m >> 32 * w + 31 & 1) * 2**32 for w in range(words)] for m in seen]
    return _i32(out)


def _unpacked(bits: torch.Tensor, n: int) -> torch.Tensor:
    j = torch.arange(n, device=DEV)
    return (bits[:, j // 32] >> (j % 32)) & 1 != 0


def _most_kids(rows: list[list[int]]) -> int:
    return max(max(parents.count(p) for p in parents) if len(parents) > 1 else 0 for parents in rows)


def _shuffled_pages(gen, lens: list[int], ppr: int, pool: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """A block table whose rows' pages lie anywhere in the pool (of ``pool`` pages, or as many as they are), and the
    pages that it leaves."""
    counts = torch.tensor([-(-n // PAGE) for n in lens], device=DEV)
    total = int(sum(-(-n // PAGE) for n in lens))
    ids = (torch.randperm(max(total, pool), generator=gen, device=DEV) + 1).to(torch.int32)
    used = torch.arange(ppr, device=DEV)[None, :] < counts[:, None]
    table = torch.zeros(len(lens), ppr, dtype=torch.int32, device=DEV)
    table[used] = ids[:total]
    return table, ids[total:]


def _ring(free_ids: torch.Tensor, cap: int, seed: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The ring of free pages, its first entry anywhere, so that it wraps around its end."""
    free = torch.zeros(cap, dtype=torch.int32, device=DEV)
    head = (seed * 7919) % cap
    free[(head + torch.arange(free_ids.numel(), device=DEV)) % cap] = free_ids
    return free, _i32([head, free_ids.numel()])


def _layers(case: dict, gen, n_pages: int) -> list[torch.Tensor]:
    """K and V pages of every layer, page 0 empty."""
    out = []
    for _ in range(2 * case["layers"]):
        x = torch.randn(n_pages + 1, case["Hkv"], PAGE, case["D"], generator=gen, device=DEV, dtype=DTYPES[case["dtype"]])
        x[0] = 0
        out.append(x)
    return out


def _tree_inputs(case: dict, seed: int) -> dict:
    rng = random.Random(seed + 1)
    rows = _trees(case, seed)
    new = [len(r) for r in rows]
    lens = [rng.randint(0, 8000) + n for n in new]
    return dict(parents=_flat(rows, 3), lens=_i32(lens), starts=_i32(_starts(new)), most=case["nodes"])


def _attend_lengths(case: dict, seed: int) -> tuple[list[int], list[list[int]]]:
    """Every row's tokens (the drafted ones included), and its tree."""
    rows = _trees(case, seed)
    held = _log_lengths(random.Random(seed), case["B"], case["Lmin"], case["Lmax"])
    return [n + len(r) for n, r in zip(held, rows)], rows


def _attend_inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    dt = DTYPES[case["dtype"]]
    lens, rows = _attend_lengths(case, seed)
    new = [len(r) for r in rows]
    table, _ = _shuffled_pages(gen, lens, max(-(-n // PAGE) for n in lens) + 3)
    n_pages = sum(-(-n // PAGE) for n in lens) + 1
    chan = torch.exp(0.5 * torch.randn(1, Hkv, 1, D, generator=gen, device=DEV))
    k = (torch.randn(n_pages, Hkv, PAGE, D, generator=gen, device=DEV) * chan).to(dt)
    v = torch.randn(n_pages, Hkv, PAGE, D, generator=gen, device=DEV).to(dt)
    k[0] = 0
    v[0] = 0
    q = torch.randn(sum(new), Hq, D, generator=gen, device=DEV).to(dt)
    bits = _sight(rows, -(-case["nodes"] // 32))  # of the step's tree, which every layer's attention takes
    s = dict(q=q, k_pages=k, v_pages=v, table=table, lens=_i32(lens), starts=_i32(_starts(new)), scale=1.0 / math.sqrt(D),
             sees=_unpacked(bits, max(new)), most_len=max(lens))
    if own:
        from fade_amd.kernels.paged import PagedAttentionPlan

        s["plan"] = PagedAttentionPlan(q, k, v, table, s["lens"], s["starts"], sm_scale=s["scale"], mask="tree", tree=bits)
    return s


def _verify_inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows = _trees(case, seed)
    new, dt, V = [len(r) for r in rows], DTYPES[case["dtype"]], case["V"]
    T, starts = sum(new), _starts(new)
    # peaked, as a language model's, and a draft's that is near them
    z = 4.5 * torch.randn(T, V, generator=gen, device=DEV)
    near = z + 0.8 * torch.randn(T, V, generator=gen, device=DEV)
    target, near = torch.softmax(z, -1).to(dt), torch.softmax(near, -1).to(dt)
    del z
    parents = _flat(rows)
    parent_row = _i32([starts[b] + max(p, 0) for b, r in enumerate(rows) for p in r]).long()
    if case["draft"]:  # drawn from the parent's draft probabilities
        pick = torch.rand(T, 1, generator=gen, device=DEV, dtype=torch.float64)
        c = near.double().cumsum(-1)
        tokens = torch.searchsorted(c[parent_row], pick * c[parent_row, -1:], right=True)[:, 0].clamp_(max=V - 1)
        del c
    else:  # a child's rank among its siblings is its rank in the draft
        rank, seen = [], {}
        for b, r in enumerate(rows):
            for p in r:
                seen[b, p] = seen.get((b, p), -1) + 1
                rank.append(seen[b, p])
        tokens = near.topk(case["fan"] + 1, dim=-1).indices[parent_row, torch.tensor(rank, device=DEV)]
    return dict(target=target, draft=near if case["draft"] else None, tokens=tokens, parents=parents, starts=_i32(starts),
                uniforms=torch.rand(T, generator=gen, device=DEV), final=torch.rand(case["B"], generator=gen, device=DEV),
                max_path=case["nodes"], most=max(new), kids=_most_kids(rows), sees=_unpacked(_sight(rows, -(-case["nodes"] // 32)), max(new)))


def _accept_lengths(case: dict, seed: int) -> tuple[list[int], list[list[int]], list[list[int]]]:
    """Every row's tokens (the drafted ones included), its tree and the accepted path in it: from the first token to
    one anywhere."""
    rng = random.Random(seed)
    rows = _trees(case, seed)
    held = _spread(rng, case["B"], 0, case["held"])
    paths = []
    for parents in rows:
        i, path = rng.randrange(len(parents)), []
        while i >= 0:
            path.append(i)
            i = parents[i]
        paths.append(path[::-1])
    return [n + len(r) for n, r in zip(held, rows)], rows, paths


def _accept_inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    lens, rows, paths = _accept_lengths(case, seed)
    ppr = -(-(case["held"] + case["nodes"]) // PAGE) + 2
    pages = sum(-(-n // PAGE) for n in _spread(random.Random(0), case["B"], 0, case["held"])) + case["B"] * -(-case["nodes"] // PAGE) + 9
    table, left = _shuffled_pages(gen, lens, ppr, pages)
    free, ring = _ring(left, pages, seed)
    return dict(path=_i32([p + [-1] * (case["nodes"] - len(p)) for p in paths]), counts=_i32([len(p) for p in paths]), table=table, lens=_i32(lens),
                starts=_i32(_starts([len(r) for r in rows])), free=free, ring=ring, pages=_layers(case, gen, pages))


def _fork_rows(case: dict, seed: int):
    """(a group's shared pages, every beam's own tokens behind them, every output row's source and kept tokens)"""
    rng = random.Random(seed)
    shared = _spread(rng, case["groups"], case["held"] // (2 * PAGE), case["held"] // PAGE)
    tokens = _spread(rng, case["groups"] * case["beams"], 1, 300)
    mine = [tokens[g * case["beams"]:(g + 1) * case["beams"]] for g in range(case["groups"])]
    source = [g * case["beams"] + rng.randrange(case["beams"]) for g in range(case["groups"]) for _ in range(case["out"])]
    keep = [WHOLE] * len(source)
    picked = rng.sample(range(len(source)), case["drops"] + case["cuts"])
    for r in picked[:case["drops"]]:
        source[r] = -1
    for r in picked[case["drops"]:]:
        g, i = divmod(source[r], case["beams"])
        keep[r] = rng.randint(0, shared[g] * PAGE + mine[g][i])
    return shared, mine, source, keep


def _fork_inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    shared, mine, source, keep = _fork_rows(case, seed)
    ppr = case["held"] // PAGE + 7
    used = sum(shared) + sum(-(-n // PAGE) for row in mine for n in row)
    cap = used + len(source) + 5
    ids = (torch.randperm(cap, generator=gen, device=DEV) + 1).to(torch.int32)
    order, at, lens, table = ids.tolist(), 0, [], []
    for n, beams in zip(shared, mine):
        prefix = order[at:at + n]
        at += n
        for tokens in beams:
            more = -(-tokens // PAGE)
            table.append(prefix + order[at:at + more] + [0] * (ppr - n - more))
            at += more
            lens.append(n * PAGE + tokens)
    free, ring = _ring(ids[used:], cap, seed)
    return dict(lens=_i32(lens), table=_i32(table), source=_i32(source), keep=_i32(keep), free=free, ring=ring, pages=_layers(case, gen, cap))


def prepare(case: dict, seed: int) -> dict:
    make = dict(tree=_tree_inputs, attend=_attend_inputs, verify=_verify_inputs, accept=_accept_inputs, fork=_fork_inputs)[case["kind"]]
    s = dict(make(case, seed), kind=case["kind"])
    if own and "pages" in s:
        from fade_amd.pages import PageLayers

        s["layers"] = PageLayers(s["pages"])  # a program makes it with its pages
    return s


# ------------------------------------------------------------- the plain forms
def _rows_of(starts, n_tokens: int):
    """Each token's row, its place among the row's new tokens, and whether it belongs to one."""
    t = torch.arange(n_tokens, device=DEV)
    live = t < starts[-1]
    row = torch.where(live, torch.searchsorted(starts[1:].contiguous(), t, right=True), 0)
    return row, torch.where(live, t - starts[row], 0), live


def _plain_tree(s: dict) -> dict:
    parents, starts, n = s["parents"].long(), s["starts"].long(), s["most"]
    row, i, live = _rows_of(starts, parents.numel())
    t = torch.arange(parents.numel(), device=DEV)
    up = torch.where(live & (parents >= 0), starts[row] + parents, t)  # a root hangs on itself
    sees = (torch.arange(n, device=DEV) == i[:, None]) & live[:, None]
    for _ in range((n - 1).bit_length()):  # what an ancestor 2, 4, 8 .. steps up sees, too
        sees, up = sees | sees[up], up[up]
    words = torch.nn.functional.pad(sees, (0, -n % 32)).view(parents.numel(), -1, 32).long() << torch.arange(32, device=DEV)
    depth = sees.sum(-1) - live.long()
    positions = torch.where(live, (s["lens"].long() - (starts[1:] - starts[:-1]))[row] + depth, 0)
    return dict(bits=words.sum(-1).int(), depth=depth.int(), positions=positions.int())


def _plain_attend(s: dict) -> torch.Tensor:
    """Rows padded to the longest one, in 32 bits."""
    q, table, lens, starts = s["q"], s["table"].long(), s["lens"].long(), s["starts"].long()
    T, Hq, D = q.shape
    Hkv = s["k_pages"].shape[1]
    B, n, pages = table.shape[0], s["sees"].shape[1], -(-s["most_len"] // PAGE)
    i = torch.arange(n, device=DEV)
    new = starts[1:] - starts[:-1]
    qi = torch.where(i < new[:, None], starts[:-1, None] + i, 0)
    qp = q.float()[qi].transpose(1, 2).reshape(B, Hkv, Hq // Hkv * n, D)
    k = s["k_pages"][table[:, :pages]].float().transpose(1, 2).reshape(B, Hkv, pages * PAGE, D)
    v = s["v_pages"][table[:, :pages]].float().transpose(1, 2).reshape(B, Hkv, pages * PAGE, D)
    x = torch.matmul(qp, k.transpose(2, 3)) * s["scale"]
    # key j of a row: before the drafted tokens, or one of them that the query sees
    j = torch.arange(pages * PAGE, device=DEV) - (lens - new)[:, None]
    drafted = torch.gather(s["sees"][qi], 2, j.clamp(0, n - 1)[:, None].expand(B, n, pages * PAGE))
    seen = (j < 0)[:, None] | ((j < new[:, None])[:, None] & drafted)
    x = x.reshape(B, Hkv, Hq // Hkv, n, pages * PAGE).masked_fill_(~seen[:, None, None], -math.inf)
    e = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(e.reshape(B, Hkv, Hq // Hkv * n, pages * PAGE), v).reshape(B, Hkv, Hq // Hkv, n, D) / e.sum(-1, keepdim=True)
    o = o.reshape(B, Hq, n, D).transpose(1, 2)
    row, place, _ = _rows_of(starts, T)
    return o[row, place].to(q.dtype)


def _plain_verify(s: dict) -> dict:
    """All tokens' tests at once, in 64 bits (sums over a vocabulary, values next to a border)."""
    target, draft, starts, n = s["target"], s["draft"], s["starts"].long(), s["most"]
    T, V = target.shape
    B, i = starts.numel() - 1, torch.arange(n, device=DEV)
    live = i < (starts[1:] - starts[:-1])[:, None]
    at = torch.where(live, starts[:-1, None] + i, 0)  # [B, n]
    parent = torch.where(live, s["parents"].long()[at], -2)
    up = starts[:-1, None] + parent.clamp(min=0)
    tok, u = s["tokens"][at], s["uniforms"].double()[at]
    p = target[up, tok].double()
    child = live & (parent >= 0)
    sibling = (parent[:, :, None] == parent[:, None, :]) & child[:, :, None] & child[:, None, :]
    earlier = sibling & (i < i[:, None])
    if draft is not None:
        # after k of a token's children are refused, what is left of its probabilities is max(p - s_k q, 0) / N_k
        shares, norms = [torch.zeros(T, 1, dtype=torch.float64, device=DEV)], [torch.ones(T, 1, dtype=torch.float64, device=DEV)]
        for _ in range(s["kids"]):
            shares.append(shares[-1] + norms[-1])
            norms.append((target.double() - shares[-1] * draft.double()).clamp_(min=0).sum(-1, keepdim=True))
        shares, norms = torch.cat(shares, 1), torch.cat(norms, 1)
        rank, q = earlier.sum(-1), draft[up, tok].double()
        left, bound = (p - shares[up, rank] * q).clamp(min=0), u * norms[up, rank] * q
    else:
        again = (earlier & (tok[:, :, None] == tok[:, None, :])).any(-1)  # a token that was refused already
        left = torch.where(again, 0.0, p)
        bound = u * (1.0 - (earlier * left[:, None, :]).sum(-1))
    ok = child & (left > 0) & (bound < left)
    chosen = ok & ~(earlier & ok[:, None, :]).any(-1)
    chosen[:, 0] |= live[:, 0]
    on_path = live & ~(s["sees"][at][..., :n] & ~chosen[:, None, :]).any(-1)
    counts = on_path.sum(-1)
    order = torch.where(on_path, on_path.cumsum(-1) - 1, s["max_path"])
    path = torch.full((B, s["max_path"] + 1), -1, dtype=torch.long, device=DEV).scatter_(1, order, i.expand(B, n))[:, :-1]
    last = torch.where(on_path, i, -1).amax(-1).clamp(min=0)
    end = starts[:-1] + last
    w = target[end].double()
    refused = child & (parent == last[:, None])
    if draft is not None:
        w = (w - shares[end, refused.sum(-1)][:, None] * draft[end].double()).clamp_(min=0)
    else:
        w = torch.nn.functional.pad(w, (0, 1)).scatter_(1, torch.where(refused, tok, V), 0.0)[:, :V]
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, target[end].double())
    c = w.cumsum(-1)
    nxt = (c <= s["final"].double()[:, None] * c[:, -1:]).sum(-1).clamp_(max=V - 1)
    # the tokens that the row goes on by: the path's behind its first, then the next one
    j = torch.arange(s["max_path"], device=DEV)
    after = torch.nn.functional.pad(path, (0, 1), value=0)[:, 1:].clamp(min=0)
    tokens = torch.where(j < counts[:, None] - 1, torch.gather(tok, 1, after), torch.where(j == counts[:, None] - 1, nxt[:, None], -1))
    return dict(path=path.int(), counts=counts.int(), tokens=tokens, next=nxt)


def _plain_compact(s: dict) -> torch.Tensor:
    lens, starts, table = s["lens"].long(), s["starts"].long(), s["table"].long()
    base = lens - (starts[1:] - starts[:-1])
    j = torch.arange(s["path"].shape[1], device=DEV)
    live = j < s["counts"][:, None]
    where = lambda pos: (torch.where(live, torch.gather(table, 1, pos // PAGE), 0), torch.where(live, pos % PAGE, 0))  # noqa: E731
    (sp, si), (dp, di) = where(base[:, None] + s["path"].clamp(min=0)), where(base[:, None] + j)
    for x in s["pages"]:
        x[dp, :, di] = x[sp, :, si]
    return (base + s["counts"]).int()


def _plain_fork(s: dict, source, keep) -> dict:
    lens, table = s["lens"].long(), s["table"]
    B, ppr = table.shape
    cap, head, count = s["free"].numel(), s["ring"][0].long(), s["ring"][1].long()
    R, col = source.numel(), torch.arange(ppr, device=DEV)
    src = source.long().clamp(min=0)
    n = torch.where(source >= 0, torch.minimum(lens[src], keep.long()), 0)
    pages = (n + PAGE - 1) // PAGE
    held = col < pages[:, None]
    new = torch.where(held, table[src], 0)
    had = col < ((lens + PAGE - 1) // PAGE)[:, None]
    before = torch.zeros(cap + 1, dtype=torch.long, device=DEV).scatter_add_(0, table.long().reshape(-1), had.long().reshape(-1))
    after = torch.zeros_like(before).scatter_add_(0, new.long().reshape(-1), held.long().reshape(-1))
    # the page that a row goes on writing: its own, so all but one of the rows that end in it (or all) get a copy
    part = n % PAGE != 0
    end = (pages - 1).clamp(min=0)
    last = torch.gather(new, 1, end[:, None])[:, 0].long()
    ends = torch.zeros_like(before).scatter_add_(0, last, part.long())
    row = torch.arange(R, device=DEV)
    first = torch.full_like(before, R).scatter_reduce_(0, last, torch.where(part, row, R), "amin")
    copied = part & ((after[last] > ends[last]) | (first[last] != row))
    fresh = s["free"][(head + copied.cumsum(0) - 1) % cap]
    new = torch.where(copied[:, None] & (col == end[:, None]), fresh[:, None], new)
    copies = torch.where(copied[:, None], torch.stack([last.int(), fresh, (n % PAGE).int()], 1), 0)
    # pages that nobody holds any more, in the order of their numbers
    left = (before > 0) & (after == 0)
    left[0] = False
    at = torch.where(left, (head + count + left.cumsum(0) - 1) % cap, cap)
    free = torch.nn.functional.pad(s["free"], (0, 1)).scatter_(0, at, torch.arange(cap + 1, dtype=torch.int32, device=DEV))
    s["free"].copy_(free[:cap])
    taken = copied.sum()
    return dict(table=new, lens=n.int(), copies=copies, ring=torch.stack([(head + taken) % cap, count - taken + left.sum()]).int(), free=s["free"])


def _plain_copy(s: dict, copies) -> None:
    live = torch.arange(PAGE, device=DEV)[None, :] < copies[:, 2:]
    src, dst = copies[:, 0].long(), copies[:, 1].long()
    for x in s["pages"]:
        x[dst] = torch.where(live[:, None, :, None], x[src], x[dst])  # (rows without a copy: page 0 to itself)


def run(s: dict):
    kind = s["kind"]
    if kind == "attend":
        return s["plan"].run() if own else _plain_attend(s)
    if kind == "tree":
        if not own:
            return _plain_tree(s)
        from fade_amd.kernels.drafts import draft_tree

        r = draft_tree(s["parents"], s["lens"], s["starts"], s["most"])
        return dict(bits=r.bits, depth=r.depth, positions=r.positions)
    if kind == "verify":
        if not own:
            return _plain_verify(s)
        from fade_amd.kernels.drafts import verify_drafts

        r = verify_drafts(s["target"], s["tokens"], s["parents"], s["starts"], s["uniforms"], s["final"], s["max_path"], draft=s["draft"])
        return dict(path=r.path, counts=r.counts, tokens=r.tokens, next=r.next)
    if kind == "accept":
        if not own:
            kept = _plain_compact(s)
            return dict(_plain_fork(s, torch.arange(kept.numel(), device=DEV), kept), pages=s["pages"])
        from fade_amd.kernels.paged import paged_compact
        from fade_amd.pages import page_fork

        kept = paged_compact(s["path"], s["counts"], s["table"], s["lens"], s["starts"], s["layers"])
        r = page_fork(s["lens"], s["table"], s["free"], s["ring"], keep=kept)
    else:
        if not own:
            r = _plain_fork(s, s["source"], s["keep"])
            _plain_copy(s, r["copies"])
            return dict(r, pages=s["pages"])
        from fade_amd.kernels.paged import paged_copy
        from fade_amd.pages import page_fork

        r = page_fork(s["lens"], s["table"], s["free"], s["ring"], source=s["source"], keep=s["keep"])
        paged_copy(r.copies, s["layers"])
    return dict(table=r.table, lens=r.lens, copies=r.copies, ring=r.ring, free=s["free"], pages=s["pages"])


# -------------------------------------------------------------------- the work
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "tree":
        T = sum(len(r) for r in _trees(case, 0)) + 3
        return {"bytes": 4.0 * (T * (3 + -(-case["nodes"] // 32)) + 2 * case["B"] + 1), "flops": 0.0}
    if kind == "verify":
        # the probabilities at a path's end; of the others two numbers a token
        size, T = 4 if case["dtype"] == "fp32" else 2, sum(len(r) for r in _trees(case, 0))
        return {"bytes": (1.0 + case["draft"]) * size * case["B"] * case["V"] + 28.0 * T, "flops": 4.0 * case["B"] * case["V"]}
    Hkv, D = case["Hkv"], case["D"]
    if kind == "attend":
        lens, rows = _attend_lengths(case, 0)
        new = [len(r) for r in rows]
        pairs = sum(n * (L - n) for L, n in zip(lens, new)) + 4.0 * sum(new)  # (a drafted token sees about three others)
        return {"bytes": 4.0 * (sum(lens) * Hkv + sum(new) * case["Hq"]) * D, "flops": 4.0 * pairs * case["Hq"] * D}
    token = 2 * case["layers"] * Hkv * D * 2  # bytes of one token in all layers
    if kind == "accept":
        lens, rows, paths = _accept_lengths(case, 0)
        moved = sum(i != x for path in paths for i, x in enumerate(path))
        pages = sum(-(-n // PAGE) for n in lens)
        return {"bytes": 2.0 * moved * token + 4.0 * (2 * pages + sum(map(len, paths))), "flops": 0.0}
    s = _fork_host(case, 0)
    return {"bytes": 2.0 * token * sum(c[2] for c in s["copies"]) + 4.0 * sum(len(r) for r in s["was"] + s["table"]), "flops": 0.0}


# -------------------------------------------------- the definitions, in 64 bits
def _exact_tree(case: dict, seed: int) -> dict:
    s, rows = _tree_inputs(case, seed), _trees(case, seed)
    lens, words = s["lens"].tolist(), -(-case["nodes"] // 32)
    bits, depth, positions = _sight(rows, words).tolist(), [], []
    for b, parents in enumerate(rows):
        d = []
        for p in parents:
            d.append(0 if p < 0 else d[p] + 1)
        depth += d
        positions += [lens[b] - len(parents) + x for x in d]
    out = dict(bits=bits + [[0] * words] * 3, depth=depth + [0] * 3, positions=positions + [0] * 3)
    return {name: torch.tensor(x, dtype=torch.int32) for name, x in out.items()}


def _exact_attend(case: dict, seed: int) -> torch.Tensor:
    """Row by row and head by head, a softmax over the visible keys."""
    s = _attend_inputs(case, seed)
    lens, rows = _attend_lengths(case, seed)
    G, at, out = case["Hq"] // case["Hkv"], 0, []
    for b, (L, parents) in enumerate(zip(lens, rows)):
        n = len(parents)
        ids = s["table"][b, :-(-L // PAGE)].long()
        q = s["q"][at:at + n].double()
        at += n
        seen = torch.zeros(n, L, dtype=torch.bool)
        seen[:, :L - n] = True
        for i, p in enumerate(parents):
            if p >= 0:
                seen[i] |= seen[p]
            seen[i, L - n + i] = True
        seen = seen.to(DEV)
        heads = []
        for h in range(case["Hkv"]):
            k, v = (s[x][ids, h].double().reshape(-1, case["D"])[:L] for x in ("k_pages", "v_pages"))
            x = torch.einsum("nge,le->gnl", q[:, h * G:(h + 1) * G], k) * s["scale"]
            heads.append(torch.softmax(x.masked_fill(~seen, -math.inf), dim=-1) @ v)
        out.append(torch.cat(heads).transpose(0, 1))
    return torch.cat(out)


def _exact_verify(case: dict, seed: int) -> dict:
    """Row by row: a walk down the tree, on distributions that are renormalized after each refusal."""
    s, rows = _verify_inputs(case, seed), _trees(case, seed)
    tokens, uniforms, final = s["tokens"].tolist(), s["uniforms"].tolist(), s["final"].tolist()
    at, width, out = 0, s["max_path"], dict(path=[], counts=[], tokens=[], next=[])
    for b, parents in enumerate(rows):
        node, path = 0, [0]
        while True:
            p = s["target"][at + node].double()
            q = s["draft"][at + node].double() if case["draft"] else None
            go = None
            for c in (i for i, x in enumerate(parents) if x == node):
                x, u = tokens[at + c], uniforms[at + c]
                if q is None:
                    if float(p[x]) > u:
                        go = c
                        break
                    # the token is ruled out, the others' probabilities grow by as much
                    out_of = float(p[x])
                    p[x] = 0.0
                    p = p / (1.0 - out_of) if out_of < 1.0 else p
                else:
                    if float(p[x]) > u * float(q[x]):
                        go = c
                        break
                    rest = (p - q).clamp(min=0)
                    p = rest / rest.sum() if float(rest.sum()) > 0 else rest
            if go is None:
                break
            node = go
            path.append(go)
        if float(p.sum()) <= 0:
            p = s["target"][at + node].double()
        c = p.cumsum(0)
        nxt = min(int(torch.searchsorted(c, c[-1:] * final[b], right=True)), case["V"] - 1)
        emitted = [tokens[at + i] for i in path[1:]] + [nxt]
        rest = [-1] * (width - len(path))
        out["path"].append(path + rest)
        out["counts"].append(len(path))
        out["tokens"].append(emitted + rest)
        out["next"].append(nxt)
        at += len(parents)
    kind = dict(path=torch.int32, counts=torch.int32, tokens=torch.int64, next=torch.int64)
    return {name: torch.tensor(x, dtype=kind[name]) for name, x in out.items()}


def _exact_accept(case: dict, seed: int) -> dict:
    s = _accept_inputs(case, seed)
    lens, rows, paths = _accept_lengths(case, seed)
    table, free, (head, count) = s["table"].tolist(), s["free"].tolist(), s["ring"].tolist()
    src, dst, left = [], [], []
    for b, (L, parents, path) in enumerate(zip(lens, rows, paths)):
        base = L - len(parents)
        slot = lambda i: table[b][i // PAGE] * PAGE + i % PAGE  # noqa: E731
        src += [slot(base + x) for x in path]
        dst += [slot(base + i) for i in range(len(path))]
        lens[b] = base + len(path)
        keep = -(-lens[b] // PAGE)
        left += [x for x in table[b][keep:] if x]
        table[b][keep:] = [0] * (len(table[b]) - keep)
    for i, x in enumerate(sorted(left)):
        free[(head + count + i) % len(free)] = x
    pages = []
    for x in s["pages"]:
        y = x.transpose(1, 2).reshape(-1, case["Hkv"], case["D"]).double()
        y[dst] = y[src]
        pages.append(y.reshape(-1, PAGE, case["Hkv"], case["D"]).transpose(1, 2))
    out = dict(table=table, lens=lens, copies=[[0, 0, 0]] * len(lens), ring=[head, count + len(left)], free=free)
    return dict({name: torch.tensor(x, dtype=torch.int32) for name, x in out.items()}, pages=pages)


def _fork_host(case: dict, seed: int, s: dict | None = None) -> dict:
    """The output rows one after the other, on the host; pages numbered here where ``s`` does not say."""
    shared, mine, source, keep = _fork_rows(case, seed)
    lens, was, n = [], [], 0
    for g, beams in enumerate(mine):
        first, n = n, n + shared[g]
        for tokens in beams:
            more = -(-tokens // PAGE)
            was.append(list(range(first + 1, first + shared[g] + 1)) + list(range(n + 1, n + more + 1)))
            n += more
            lens.append(shared[g] * PAGE + tokens)
    if s is None:
        order = list(range(n + 1, n + len(source) + 6))
    else:
        free, (head, count) = s["free"].tolist(), s["ring"].tolist()
        was = [row[:len(x)] for row, x in zip(s["table"].tolist(), was)]
        order = [free[(head + i) % len(free)] for i in range(count)]
    table = [was[b][:-(-min(k, lens[b]) // PAGE)] if b >= 0 else [] for b, k in zip(source, keep)]
    kept = [min(k, lens[b]) if b >= 0 else 0 for b, k in zip(source, keep)]
    held: dict[int, list[int]] = {}
    for r, row in enumerate(table):
        for x in row:
            held.setdefault(x, []).append(r)
    copies, taken = [[0, 0, 0] for _ in source], 0
    new = [list(row) for row in table]
    for r, row in enumerate(table):
        if kept[r] % PAGE:
            rows = held[row[-1]]  # the first of them stays, if all end in this page
            if not (rows[0] == r and all(table[x][-1] == row[-1] and kept[x] % PAGE for x in rows)):
                copies[r] = [row[-1], order[taken], kept[r] % PAGE]
                new[r][-1] = order[taken]
                taken += 1
    left = sorted({x for row in was for x in row} - set(held))
    return dict(was=was, table=new, lens=kept, copies=copies, taken=taken, left=left)


def _exact_fork(case: dict, seed: int) -> dict:
    s = _fork_inputs(case, seed)
    r = _fork_host(case, seed, s)
    ppr, free, (head, count) = s["table"].shape[1], s["free"].tolist(), s["ring"].tolist()
    for i, x in enumerate(r["left"]):
        free[(head + count + i) % len(free)] = x
    pages = []
    for x in s["pages"]:
        y = x.double()
        for src, dst, n in r["copies"]:
            y[dst, :, :n] = y[src, :, :n]
        pages.append(y)
    out = dict(table=[row + [0] * (ppr - len(row)) for row in r["table"]], lens=r["lens"], copies=r["copies"],
               ring=[(head + r["taken"]) % len(free), count - r["taken"] + len(r["left"])], free=free)
    return dict({name: torch.tensor(x, dtype=torch.int32) for name, x in out.items()}, pages=pages)


def exact(case: dict, seed: int):
    return dict(tree=_exact_tree, attend=_exact_attend, verify=_exact_verify, accept=_exact_accept, fork=_exact_fork)[case["kind"]](case, seed)
