"""Operators of the paged 16-bit KV cache that are timed: a serving step before the compression.

Four kinds of work, each through the entry point that a serving program calls:

  slots    ``page_slots``: from every row's held and new token counts, the block
           table, the slot of each new token and the free pages, on the GPU
  rope     ``rope_axes``: q and k rotated at positions of several axes (time,
           height, width), as a vision-language model's tokens have
  append   ``paged_append``: the new tokens' k rotated and written with v into
           their pages, q rotated in the same call
  attend   ``PagedAttentionPlan``: each row's chunk of new tokens (any length, one
           included) over the row's pages

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
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# query heads, kv heads, head_dim: 8B-class GQA-4, Qwen2.5-7B's GQA-7, a 70B-class
# GQA-8, Qwen2.5-0.5B's 14/2 at head_dim 64, Gemma's 16/8 at head_dim 256
SHAPES = ((32, 8, 128), (28, 4, 128), (64, 8, 128), (14, 2, 64), (16, 8, 256))
THETA = 1.0e6
# bounds of one case's size: elements of the K pages, attention's operations, rotated elements
MOST_PAGED = 16 * 8 * 8192 * 128
MOST_FLOPS = 6.0e11
MOST_ROTATED = 16384 * 40 * 128
MOST_SCORES = 1.1e10  # the plain form's padded scores


# ------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one decoding step of a small batch: a call of a few hundred numbers, latency only
        dict(name="slots_b16_step", kind="slots", B=16, ppr=512, held=8192, chunks=0, chunk=1, resets=0),
        # a large server's step: most rows decode, some bring a piece of their prompt, finished rows are replaced
        dict(name="slots_b1000_mixed", kind="slots", B=1000, ppr=1024, held=65000, chunks=16, chunk=2048, resets=40),
        # one picture with its question: 1000-odd tokens whose positions have three axes
        dict(name="rope_image_1k", kind="rope", B=1, S=1187, Hq=28, Hkv=4, D=128, rot=128, interleaved=False, far=0, dtype="bf16"),
        # a long video in one prompt, interleaved axes, half of each head rotated
        dict(name="rope_video_16k", kind="rope", B=1, S=16384, Hq=32, Hkv=8, D=128, rot=64, interleaved=True, far=20000, dtype="fp16"),
        # the decoding step's 32 tokens into their pages
        dict(name="append_b32_step", kind="append", B=32, new=1, held=1000, Hq=64, Hkv=8, D=128, rot=128, axes=1, far=0, dtype="bf16"),
        # prompt pieces of five rows, 256 to 4096 tokens each, positions of three axes
        dict(name="append_chunks_5", kind="append", B=5, new=4096, held=700, Hq=32, Hkv=8, D=128, rot=128, axes=3, far=0, dtype="fp16"),
        # one chat sequence on a small model: latency and launches are what counts
        dict(name="attend_b1_d64", kind="attend", B=1, Hq=14, Hkv=2, D=64, Lmin=1000, Lmax=1000, new=1, chunks=0, chunk=1, mask="bottom_right", dtype="fp16"),
        # the headline workload's layer before its compression: a batch of 16 at 8K tokens
        dict(name="attend_b16_8k", kind="attend", B=16, Hq=32, Hkv=8, D=128, Lmin=8192, Lmax=8192, new=1, chunks=0, chunk=1, mask="bottom_right", dtype="fp16"),
        # a server's decoding step: rows from short to very long, 7 query heads per kv head
        dict(name="attend_ragged_bf16", kind="attend", B=61, Hq=28, Hkv=4, D=128, Lmin=190, Lmax=32000, new=1, chunks=0, chunk=1, mask="bottom_right", dtype="bf16"),
        # the same kind of step with two rows that bring a piece of their prompt
        dict(name="attend_mixed_bf16", kind="attend", B=32, Hq=64, Hkv=8, D=128, Lmin=500, Lmax=9000, new=1, chunks=2, chunk=512, mask="bottom_right", dtype="bf16"),
        # prompts in chunks of very different lengths over what the rows already hold
        dict(name="attend_chunks_fp16", kind="attend", B=8, Hq=32, Hkv=8, D=128, Lmin=2000, Lmax=9000, new=1, chunks=8, chunk=2048, mask="bottom_right", dtype="fp16"),
        # whole prompts of odd lengths at head_dim 256
        dict(name="attend_prompts_d256", kind="attend", B=3, Hq=16, Hkv=8, D=256, Lmin=1, Lmax=1, new=1, chunks=3, chunk=2999, mask="bottom_right", dtype="bf16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng) -> dict:
    kind = rng.choice(("slots", "rope", "append", "append", "attend", "attend", "attend", "attend"))
    Hq, Hkv, D = rng.choice(SHAPES[:1] * 2 + SHAPES)
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "slots":
        B, ppr = _log_int(rng, 1, 1000), _log_int(rng, 8, 1024)
        return dict(kind=kind, B=B, ppr=ppr, held=rng.randint(1, ppr * PAGE - 1), chunks=rng.randint(0, min(B, 16)),
                    chunk=_log_int(rng, 1, min(2048, ppr * PAGE)), resets=rng.randint(0, B // 4))
    rot = rng.choice((D, D, D // 2))
    far = rng.choice((0, 0, _log_int(rng, 1000, 1000000)))
    if kind == "rope":
        S = _log_int(rng, 1, MOST_ROTATED // ((Hq + Hkv) * D))
        B = max(1, min(rng.choice((1, 1, 2, 7)), MOST_ROTATED // ((Hq + Hkv) * D * S)))
        return dict(kind=kind, B=B, S=S, Hq=Hq, Hkv=Hkv, D=D, rot=rot, interleaved=rng.choice((False, True)), far=far,
                    dtype=rng.choice((dtype, dtype, "fp32")) if S < 4000 else dtype)
    if kind == "append":
        B = _log_int(rng, 1, 64)
        new = rng.choice((1, _log_int(rng, 1, max(1, MOST_ROTATED // (2 * (Hq + 2 * Hkv) * D * B)))))
        return dict(kind=kind, B=B, new=new, held=rng.randint(0, 1000), Hq=Hq, Hkv=Hkv, D=D, rot=rot, axes=rng.choice((1, 3)),
                    far=far, dtype=dtype)
    B = _log_int(rng, 1, 64)
    Lmax = _log_int(rng, 16, max(16, min(32000, MOST_PAGED // (B * Hkv * D))))
    chunks = rng.choice((0, 0, rng.randint(0, B), B))
    most = min(MOST_FLOPS / (4.0 * Hq * D * max(1, chunks)), MOST_SCORES / (B * Hq)) / (Lmax + 2048)
    chunk = _log_int(rng, 2, max(2, min(2048, int(most))))
    return dict(kind=kind, B=B, Hq=Hq, Hkv=Hkv, D=D, Lmin=max(1, Lmax // rng.choice((1, 4, 100))), Lmax=Lmax,
                new=rng.choice((1, 1, 1, 4)), chunks=chunks, chunk=chunk, mask=rng.choice(("bottom_right", "bottom_right", "bottom_right", "none")),
                dtype=dtype)


# ----------------------------------------------------------------- the inputs
def _log_lengths(rng, n: int, lo: int, hi: int) -> list[int]:
    """n lengths spread evenly over the logarithm of lo..hi, in an order of the seed's."""
    if n == 1:
        return [hi]
    out = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    rng.shuffle(out)
    return out


def _chunk_lengths(rng, n: int, most: int) -> list[int]:
    """n chunk lengths from most / 16 to most."""
    return _log_lengths(rng, n, max(1, most // 16), most) if n else []


def _starts(new: list[int]) -> list[int]:
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _i32(x) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _shuffled_pages(gen, lens: list[int], ppr: int) -> tuple[torch.Tensor, int]:
    """A block table whose rows' pages lie anywhere in the pool, and the pool's pages (the zero page first)."""
    counts = torch.tensor([-(-n // PAGE) for n in lens], device=DEV)
    total = int(sum(-(-n // PAGE) for n in lens))
    ids = torch.randperm(total, generator=gen, device=DEV) + 1
    col = torch.arange(ppr, device=DEV)
    used = col[None, :] < counts[:, None]
    table = torch.zeros(len(lens), ppr, dtype=torch.int32, device=DEV)
    table[used] = ids.to(torch.int32)
    return table, total + 1


def _slots_lengths(case: dict, seed: int) -> tuple[list[int], list[int], list[int]]:
    rng = random.Random(seed)
    B, cap = case["B"], case["ppr"] * PAGE
    lens = [rng.randint(0, case["held"]) for _ in range(B)]
    new = [1] * B
    for b, n in zip(rng.sample(range(B), case["chunks"]), _chunk_lengths(rng, case["chunks"], case["chunk"])):
        new[b] = n
    reset = [0] * B
    for b in rng.sample(range(B), case["resets"]):
        reset[b] = 1
    lens = [min(n, cap - k) for n, k in zip(lens, new)]
    return lens, new, reset


def _slots_inputs(case: dict, seed: int) -> dict:
    lens, new, reset = _slots_lengths(case, seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    table, used = _shuffled_pages(gen, lens, case["ppr"])
    cap = (case["B"] + case["resets"]) * case["ppr"] + 7
    ids = torch.randperm(cap - used + 1, generator=gen, device=DEV).to(torch.int32) + used
    free = torch.zeros(cap, dtype=torch.int32, device=DEV)
    head = (seed * 7919) % cap  # anywhere on the ring, so that the free pages wrap around its end
    free[(head + torch.arange(ids.numel(), device=DEV)) % cap] = ids
    return dict(lens=_i32(lens), new=_i32(new), reset=torch.tensor(reset, dtype=torch.bool, device=DEV), table=table,
                free=free, ring=_i32([head, ids.numel()]), n_tokens=sum(new) + 13)


def _sections(rot: int, interleaved: bool) -> list[int]:
    """Frequencies of the time, height and width axes: 16, 24, 24 of 64, or interleaved 24, 20, 20."""
    n = rot // 2
    side = 5 * n // 16 if interleaved else 3 * n // 8
    return [n - 2 * side, side, side]


def _inv_freq(rot: int) -> torch.Tensor:
    """1 / theta ** (2 i / rot) in fp32, on the host."""
    return 1.0 / (THETA ** (torch.arange(0, rot, 2, dtype=torch.float32) / rot))


def _axis_of(rot: int, interleaved: bool) -> list[int]:
    sec = _sections(rot, interleaved)
    if not interleaved:
        return [0] * sec[0] + [1] * sec[1] + [2] * sec[2]
    return [i % 3 if i < 3 * sec[i % 3] else 0 for i in range(rot // 2)]


def _grid_positions(n: int, far: int) -> torch.Tensor:
    """[3, n]: text, then frames of 24 x 32 patches, as a vision-language prompt has them."""
    t = torch.arange(n, device=DEV)
    text = min(n, 40)
    p = t - text
    frame, y, x = p // 768, (p % 768) // 32, p % 32
    grid = torch.stack([text + frame, text + y, text + x])
    return torch.where(t[None, :] < text, t[None, :].expand(3, n), grid) + far


def _scheme(case: dict):
    """The rotary scheme a program keeps (None for the plain form)."""
    if not own:
        return None
    from fade_amd.rope import MRope, Vanilla

    if case.get("axes", 3) == 1 and case["rot"] == case["D"]:
        return Vanilla(theta=THETA, head_dim=case["D"])
    return MRope(theta=THETA, head_dim=case["D"], partial_rotary_factor=case["rot"] / case["D"],
                 mrope_section=_sections(case["rot"], case.get("interleaved", False)), interleaved=case.get("interleaved", False))


def _rope_inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, S, D = case["B"], case["S"], case["D"]
    dt = DTYPES[case["dtype"]]
    # as the projections leave them: [B, S, heads, D], seen as [B, heads, S, D]
    q = torch.randn(B, S, case["Hq"], D, generator=gen, device=DEV).to(dt).transpose(1, 2)
    k = torch.randn(B, S, case["Hkv"], D, generator=gen, device=DEV).to(dt).transpose(1, 2)
    pos = torch.stack([_grid_positions(S, case["far"] + (seed % 97) + 31 * b) for b in range(B)], dim=1)
    return dict(q=q, k=k, positions=pos, inv=_inv_freq(case["rot"]).to(DEV),
                axis=torch.tensor(_axis_of(case["rot"], case["interleaved"]), device=DEV), scheme=_scheme(case))


def _append_inputs(case: dict, seed: int) -> dict:
    rng = random.Random(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    dt = DTYPES[case["dtype"]]
    held = [rng.randint(0, case["held"]) for _ in range(B)]
    new = [1] * B if case["new"] == 1 else _chunk_lengths(rng, B, case["new"])
    after = [h + n for h, n in zip(held, new)]
    most = -(-(case["held"] + case["new"]) // PAGE)
    table, n_pages = _shuffled_pages(gen, after, most)[0], B * most + 1
    T, pad = sum(new), 5  # a few places behind the last sequence
    row = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(new, device=DEV))
    pos = torch.arange(T, device=DEV) - _i32(_starts(new)).long()[row] + torch.tensor(held, device=DEV)[row]
    slots = torch.full((T + pad,), -1, dtype=torch.int32, device=DEV)
    slots[:T] = (table.long()[row, pos // PAGE] * PAGE + pos % PAGE).to(torch.int32)
    # one projection's output, q | k | v side by side
    qkv = torch.randn(T + pad, Hq + 2 * Hkv, D, generator=gen, device=DEV).to(dt)
    p = torch.zeros(T + pad, dtype=torch.long, device=DEV)
    p[:T] = pos + case["far"]
    if case["axes"] == 3:
        p = p[None, :] + torch.stack([torch.zeros_like(p), torch.arange(T + pad, device=DEV) // 32 % 24, torch.arange(T + pad, device=DEV) % 32])
    pages = [torch.randn(n_pages, Hkv, PAGE, D, generator=gen, device=DEV).to(dt) for _ in range(2)]
    for x in pages:
        x[0] = 0
    axis = _axis_of(case["rot"], False) if case["axes"] == 3 else [0] * (case["rot"] // 2)
    return dict(q=qkv[:, :Hq], k=qkv[:, Hq:Hq + Hkv], v=qkv[:, Hq + Hkv:], k_pages=pages[0], v_pages=pages[1], slots=slots,
                n=T, positions=p, inv=_inv_freq(case["rot"]).to(DEV), axis=torch.tensor(axis, device=DEV), scheme=_scheme(case))


def _attend_lengths(case: dict, seed: int) -> tuple[list[int], list[int]]:
    """Every row's tokens (its new ones included) and its new tokens."""
    rng = random.Random(seed)
    B = case["B"]
    held = _log_lengths(rng, B, case["Lmin"], case["Lmax"])
    new = [min(case["new"], n) for n in held]
    for b, n in zip(rng.sample(range(B), case["chunks"]), _chunk_lengths(rng, case["chunks"], case["chunk"])):
        held[b] += n - new[b]
        new[b] = n
    return held, new


def _attend_inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    dt = DTYPES[case["dtype"]]
    lens, new = _attend_lengths(case, seed)
    ppr = max(-(-n // PAGE) for n in lens) + 3
    table, n_pages = _shuffled_pages(gen, lens, ppr)
    chan = torch.exp(0.5 * torch.randn(1, Hkv, 1, D, generator=gen, device=DEV))
    k = (torch.randn(n_pages, Hkv, PAGE, D, generator=gen, device=DEV) * chan).to(dt)
    v = torch.randn(n_pages, Hkv, PAGE, D, generator=gen, device=DEV).to(dt)
    k[0] = 0
    v[0] = 0
    q = torch.randn(sum(new), Hq, D, generator=gen, device=DEV).to(dt)
    s = dict(q=q, k_pages=k, v_pages=v, table=table, lens=_i32(lens), starts=_i32(_starts(new)), scale=1.0 / math.sqrt(D),
             most_new=max(new), most_len=max(lens), mask=case["mask"])
    if own:
        from fade_amd.kernels.paged import PagedAttentionPlan

        s["plan"] = PagedAttentionPlan(q, k, v, table, s["lens"], s["starts"], sm_scale=s["scale"], mask=case["mask"])
    return s


def prepare(case: dict, seed: int) -> dict:
    make = dict(slots=_slots_inputs, rope=_rope_inputs, append=_append_inputs, attend=_attend_inputs)[case["kind"]]
    return dict(make(case, seed), kind=case["kind"])


# ------------------------------------------------------------- the plain forms
def _plain_slots(s: dict) -> dict:
    held = torch.where(s["reset"], 0, s["lens"]).long()
    after = held + s["new"]
    have, old = (held + PAGE - 1) // PAGE, (s["lens"].long() + PAGE - 1) // PAGE
    need = (after + PAGE - 1) // PAGE - have
    cap, head, count = s["free"].numel(), s["ring"][0].long(), s["ring"][1].long()
    base = torch.cumsum(need, 0) - need
    starts = torch.nn.functional.pad(torch.cumsum(s["new"], 0), (1, 0))
    col = torch.arange(s["table"].shape[1], device=DEV)
    fresh = (col >= have[:, None]) & (col < (have + need)[:, None])
    place = (head + (base - have)[:, None] + col) % cap
    table = torch.where(fresh, s["free"][place], torch.where(col < have[:, None], s["table"], 0))
    # the pages of rows that start anew go behind the free ones
    back = torch.where(s["reset"], old, 0)
    at = (head + count + (torch.cumsum(back, 0) - back)[:, None] + col) % cap
    ext = torch.nn.functional.pad(s["free"], (0, 1))
    ext[torch.where(col < back[:, None], at, cap)] = s["table"]  # (the others to a place that is dropped)
    s["free"].copy_(ext[:cap])
    ring = torch.stack([(head + need.sum()) % cap, count - need.sum() + back.sum()])
    t = torch.arange(s["n_tokens"], device=DEV)
    row = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    live = t < starts[-1]
    row = torch.where(live, row, 0)
    pos = torch.where(live, held[row] + t - starts[row], 0)
    slot = torch.where(live, table[row, pos // PAGE].long() * PAGE + pos % PAGE, -1)
    return dict(table=table, lens=after.int(), starts=starts.int(), slots=slot.int(), positions=pos.int(), ring=ring.int(), free=s["free"])


def _plain_cos_sin(positions, inv, axis):
    """cos and sin [..., frequencies]: angles in 64 bits (far positions), then 32."""
    angle = positions.double()[axis].movedim(0, -1) * inv.double()
    return angle.cos().float(), angle.sin().float()


def _plain_rotate(x, cos, sin):
    half = cos.shape[-1]
    f = x.float()
    a, b = f[..., :half], f[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, f[..., 2 * half:]], dim=-1).to(x.dtype)


def _plain_rope(s: dict) -> tuple:
    cos, sin = _plain_cos_sin(s["positions"], s["inv"], s["axis"])  # [B, S, frequencies]
    return _plain_rotate(s["q"], cos[:, None], sin[:, None]), _plain_rotate(s["k"], cos[:, None], sin[:, None])


def _plain_append(s: dict) -> dict:
    pos = s["positions"] if s["positions"].dim() == 2 else s["positions"][None]
    cos, sin = _plain_cos_sin(pos, s["inv"], s["axis"])  # [T, frequencies]
    q = _plain_rotate(s["q"], cos[:, None], sin[:, None])
    k = _plain_rotate(s["k"], cos[:, None], sin[:, None])
    slots = s["slots"][:s["n"]].long()  # the places behind them hold no token
    s["k_pages"][slots // PAGE, :, slots % PAGE] = k[:s["n"]]
    s["v_pages"][slots // PAGE, :, slots % PAGE] = s["v"][:s["n"]]
    return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])


def _plain_attend(s: dict) -> torch.Tensor:
    """Rows padded to the longest one, in 32 bits."""
    q, table, lens, starts = s["q"], s["table"].long(), s["lens"].long(), s["starts"].long()
    T, Hq, D = q.shape
    Hkv = s["k_pages"].shape[1]
    B, n, pages = table.shape[0], s["most_new"], -(-s["most_len"] // PAGE)
    i = torch.arange(n, device=DEV)
    new = starts[1:] - starts[:-1]
    qi = torch.where(i < new[:, None], starts[:-1, None] + i, 0)
    qp = q.float()[qi].transpose(1, 2).reshape(B, Hkv, Hq // Hkv * n, D)
    k = s["k_pages"][table[:, :pages]].float().transpose(1, 2).reshape(B, Hkv, pages * PAGE, D)
    v = s["v_pages"][table[:, :pages]].float().transpose(1, 2).reshape(B, Hkv, pages * PAGE, D)
    x = torch.matmul(qp, k.transpose(2, 3)) * s["scale"]
    limit = (lens - new)[:, None] + i if s["mask"] == "bottom_right" else (lens - 1)[:, None].expand(B, n)
    seen = torch.arange(pages * PAGE, device=DEV) <= limit[:, :, None]
    x = x.reshape(B, Hkv, Hq // Hkv, n, pages * PAGE).masked_fill_(~seen[:, None, None], -math.inf)
    e = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(e.reshape(B, Hkv, Hq // Hkv * n, pages * PAGE), v).reshape(B, Hkv, Hq // Hkv, n, D) / e.sum(-1, keepdim=True)
    o = o.reshape(B, Hq, n, D).transpose(1, 2)
    t = torch.arange(T, device=DEV)
    row = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return o[row, t - starts[row]].to(q.dtype)


def run(s: dict):
    kind = s["kind"]
    if not own:
        return dict(slots=_plain_slots, rope=_plain_rope, append=_plain_append, attend=_plain_attend)[kind](s)
    if kind == "attend":
        return s["plan"].run()
    if kind == "slots":
        from fade_amd.pages import page_slots

        r = page_slots(s["lens"], s["new"], s["table"], s["free"], s["ring"], s["n_tokens"], reset=s["reset"])
        return dict(table=r.table, lens=r.lens, starts=r.starts, slots=r.slots, positions=r.positions, ring=r.ring, free=s["free"])
    if kind == "rope":
        from fade_amd.rope import rope_axes

        return rope_axes(s["q"], s["k"], s["positions"], s["scheme"])
    from fade_amd.kernels.paged import paged_append

    q = paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], q=s["q"], positions=s["positions"], scheme=s["scheme"])
    return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])


# -------------------------------------------------------------------- the work
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "slots":
        lens, new, reset = _slots_lengths(case, 0)
        own_pages = sum(-(-n // PAGE) for n in lens)
        B, T = case["B"], sum(new) + 13
        # the rows' pages read, the whole table written, counts, slots and positions
        return {"bytes": 4.0 * (own_pages + B * case["ppr"] + 4 * B + 2 * T), "flops": 0.0}
    size = 4 if case["dtype"] == "fp32" else 2
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if kind == "rope":
        n = case["B"] * case["S"]
        return {"bytes": n * (2.0 * (Hq + Hkv) * D * size + 24), "flops": 3.0 * n * (Hq + Hkv) * case["rot"]}
    if kind == "append":
        new = [1] * case["B"] if case["new"] == 1 else _chunk_lengths(random.Random(0), case["B"], case["new"])
        n = sum(new) + 5
        return {"bytes": n * (2.0 * (Hq + 2 * Hkv) * D * size + 8 * case["axes"] + 4), "flops": 3.0 * n * (Hq + Hkv) * case["rot"]}
    lens, new = _attend_lengths(case, 0)
    if case["mask"] == "bottom_right":
        pairs = sum(n * (L - n) + n * (n + 1) / 2.0 for L, n in zip(lens, new))
    else:
        pairs = sum(float(n) * L for L, n in zip(lens, new))
    return {"bytes": 2.0 * size * (sum(lens) * Hkv + sum(new) * Hq) * D, "flops": 4.0 * pairs * Hq * D}


# -------------------------------------------------- the definitions, in 64 bits
def _exact_slots(case: dict, seed: int) -> dict:
    """The allocation one token after the other, on the host."""
    s = _slots_inputs(case, seed)
    lens, new, reset = _slots_lengths(case, seed)
    table, free = s["table"].tolist(), s["free"].tolist()
    head, count = s["ring"].tolist()
    cap, tail = len(free), head + count
    taken, slots, positions, starts = 0, [], [], [0]
    for b, row in enumerate(table):
        held = lens[b]
        if reset[b]:
            for j in range(-(-held // PAGE)):
                free[tail % cap] = row[j]
                tail += 1
            row[:] = [0] * len(row)
            held = 0
        for t in range(held, held + new[b]):
            if t % PAGE == 0:
                row[t // PAGE] = None  # a page of its own, named below
                taken += 1
            positions.append(t)
        lens[b] = held + new[b]
        starts.append(len(positions))
    # the pages taken, in the order in which the tokens asked for them
    first = s["free"].tolist()
    order = iter(first[(head + j) % cap] for j in range(taken))
    for b, row in enumerate(table):
        for j, x in enumerate(row):
            if x is None:
                row[j] = next(order)
        slots += [row[t // PAGE] * PAGE + t % PAGE for t in positions[starts[b]:starts[b + 1]]]
    rest = s["n_tokens"] - len(slots)
    out = dict(table=table, lens=lens, starts=starts, slots=slots + [-1] * rest, positions=positions + [0] * rest,
               ring=[(head + taken) % cap, tail - head - taken], free=free)
    return {name: torch.tensor(x, dtype=torch.int32) for name, x in out.items()}


def _exact_rotation(x: torch.Tensor, positions: torch.Tensor, case: dict, axis: list[int]) -> torch.Tensor:
    """x [tokens, heads, D] as complex numbers turned by their angles; positions [axes, tokens]."""
    half = case["rot"] // 2
    angle = torch.stack([positions[a].double() * float(f) for a, f in zip(axis, _inv_freq(case["rot"]).tolist())], dim=-1)
    z = torch.complex(x[..., :half].double(), x[..., half:2 * half].double()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    return torch.cat([z.real, z.imag, x[..., 2 * half:].double()], dim=-1)


def _exact_rope(case: dict, seed: int) -> tuple:
    s = _rope_inputs(case, seed)
    axis = _axis_of(case["rot"], case["interleaved"])
    rows = lambda x: torch.stack([_exact_rotation(x[b].transpose(0, 1), s["positions"][:, b], case, axis).transpose(0, 1)  # noqa: E731
                                  for b in range(case["B"])])
    return rows(s["q"]), rows(s["k"])


def _exact_append(case: dict, seed: int) -> dict:
    s = _append_inputs(case, seed)
    pos = s["positions"] if case["axes"] == 3 else s["positions"][None]
    axis = _axis_of(case["rot"], False) if case["axes"] == 3 else [0] * (case["rot"] // 2)
    k = _exact_rotation(s["k"], pos, case, axis)
    kp, vp = (s[x].double().transpose(1, 2).reshape(-1, case["Hkv"], case["D"]).clone() for x in ("k_pages", "v_pages"))
    n = int((s["slots"] >= 0).sum())
    kp[s["slots"][:n].long()], vp[s["slots"][:n].long()] = k[:n], s["v"][:n].double()
    paged = lambda x: x.reshape(-1, PAGE, case["Hkv"], case["D"]).transpose(1, 2)  # noqa: E731
    return dict(q=_exact_rotation(s["q"], pos, case, axis), k_pages=paged(kp), v_pages=paged(vp))


def _exact_attend(case: dict, seed: int) -> torch.Tensor:
    """Row by row and head by head, a softmax over the visible keys."""
    s = _attend_inputs(case, seed)
    lens, new = _attend_lengths(case, seed)
    G, at, out = case["Hq"] // case["Hkv"], 0, []
    for b, (L, n) in enumerate(zip(lens, new)):
        ids = s["table"][b, :-(-L // PAGE)].long()
        q = s["q"][at:at + n].double()
        at += n
        seen = torch.ones(n, L, dtype=torch.bool, device=DEV)
        if case["mask"] == "bottom_right":
            seen = seen.tril(L - n)
        heads = []
        for h in range(case["Hkv"]):
            k, v = (s[x][ids, h].double().reshape(-1, case["D"])[:L] for x in ("k_pages", "v_pages"))
            x = torch.einsum("nge,le->gnl", q[:, h * G:(h + 1) * G], k) * s["scale"]
            heads.append(torch.softmax(x.masked_fill(~seen, -math.inf), dim=-1) @ v)
        out.append(torch.cat(heads).transpose(0, 1))
    return torch.cat(out)


def exact(case: dict, seed: int):
    return dict(slots=_exact_slots, rope=_exact_rope, append=_exact_append, attend=_exact_attend)[case["kind"]](case, seed)
