"""The paged 16-bit cache on the GPU: ``page_slots`` against an allocation on the host, ``rope_axes``
and ``paged_append`` against rotations in 64 bits, ``paged_attention`` against a softmax in 64 bits,
and a run of them together as a serving step uses them."""

from __future__ import annotations

import math
import random

import pytest
import torch

from fade_amd import _lib
from fade_amd.kernels import PagedAttentionPlan, paged_append, paged_attention, tiered_prefill_attention
from fade_amd.pages import PAGE_TOKENS, MiddlePagePool, PageSlots, TokenPagePool, page_slots
from fade_amd.quant import quant_k_int4, quant_v_int4
from fade_amd.rope import LinearScaled, Llama3, MRope, NoRope, Proportional, Vanilla, Yarn, rope_axes

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------ page_slots
class _Model:
    """The free ring, the table and the rows on the host."""

    def __init__(self, n_pages, B, ppr, head=0):
        self.free = [0] * n_pages
        for j in range(n_pages):
            self.free[(head + j) % n_pages] = j + 1
        self.head, self.count = head, n_pages
        self.table = [[0] * ppr for _ in range(B)]
        self.lens = [0] * B

    def step(self, new, n_tokens, reset):
        cap, ppr = len(self.free), len(self.table[0])
        held = [0 if r else n for n, r in zip(self.lens, reset)]
        pg = lambda n: -(-n // PAGE_TOKENS)  # noqa: E731
        need = [pg(h + n) - pg(h) for h, n in zip(held, new)]
        status = 0
        if any(h + n > ppr * PAGE_TOKENS for h, n in zip(held, new)):
            status |= 2
            need = [0 if h + n > ppr * PAGE_TOKENS else k for h, n, k in zip(held, new, need)]
        fits = [0 if h + n > ppr * PAGE_TOKENS else n for h, n in zip(held, new)]
        status |= 1 if sum(need) > self.count else 0
        status |= 4 if sum(fits) > n_tokens else 0
        if status:
            return dict(status=[status], table=self.table, lens=self.lens, starts=[0] * (len(new) + 1), slots=[-1] * n_tokens,
                        positions=[0] * n_tokens, ring=[self.head, self.count])
        tail, back, slots, pos, starts = self.head + self.count, 0, [], [], [0]
        for b, row in enumerate(self.table):
            if reset[b]:
                for j in range(pg(self.lens[b])):
                    self.free[(tail + back) % cap] = row[j]
                    back += 1
                row[:] = [0] * ppr
            for j in range(pg(held[b]), pg(held[b]) + need[b]):
                row[j] = self.free[self.head]
                self.head = (self.head + 1) % cap
                self.count -= 1
            for t in range(held[b], held[b] + new[b]):
                slots.append(row[t // PAGE_TOKENS] * PAGE_TOKENS + t % PAGE_TOKENS)
                pos.append(t)
            self.lens[b] = held[b] + new[b]
            starts.append(len(slots))
        self.count += back
        rest = n_tokens - len(slots)
        return dict(status=[0], table=self.table, lens=self.lens, starts=starts, slots=slots + [-1] * rest, positions=pos + [0] * rest,
                    ring=[self.head, self.count])


def _same(got: PageSlots, want: dict, free, model):
    for name, x in want.items():
        assert getattr(got, name).tolist() == x, name
    assert free.tolist() == model.free


@pytest.mark.parametrize("B,ppr,pages", [(1, 1, 1), (1, 7, 5), (3, 5, 11), (64, 4, 200), (256, 3, 500), (257, 3, 500), (1000, 9, 6000), (4096, 2, 5000)])
def test_slots_against_the_host(dev, B, ppr, pages):
    rng = random.Random(B * 31 + ppr)
    m = _Model(pages, B, ppr, head=rng.randrange(pages))
    free, ring = _i32(m.free, dev), _i32([m.head, m.count], dev)
    lens, table = _i32(m.lens, dev), _i32(m.table, dev)
    done = 0
    for step in range(12):
        new = [rng.choice((0, 1, 1, 1, 2, 63, 64, 65)) if B < 500 else rng.choice((0, 0, 1, 1, 70)) for _ in range(B)]
        reset = [rng.random() < 0.2 for _ in range(B)]
        n = max(0, sum(new) - (1 if step == 5 else -3))
        before, ring_before, free_before = table.clone(), ring.clone(), free.clone()
        args = (lens, _i32(new, dev), table, free, ring, n)
        got = page_slots(*args, reset=torch.tensor(reset, device=dev))
        want = m.step(new, n, reset)
        _same(got, want, free, m)
        # the inputs stand, and the same inputs give the same results again
        assert torch.equal(table, before) and torch.equal(ring, ring_before)
        again = page_slots(*args, reset=torch.tensor(reset, device=dev).to(torch.uint8))
        _same(again, want, free, m)
        if want["status"] != [0]:
            assert torch.equal(free, free_before)
            with pytest.raises(RuntimeError, match="nothing was changed"):
                got.check()
        else:
            done += 1
            got.check()
        lens, table, ring = got.lens, got.table, got.ring
    assert done or pages == 1


def test_slots_in_place_table_and_without_reset(dev):
    m = _Model(40, 4, 6)
    free, ring, lens, table = _i32(m.free, dev), _i32([0, 40], dev), _i32(m.lens, dev), _i32(m.table, dev)
    for new in ([1, 64, 0, 200], [1, 1, 1, 1], [63, 0, 65, 100]):
        z = lambda n: torch.full((n,), 77, dtype=torch.int32, device=dev)  # noqa: E731
        n = sum(new)
        out = PageSlots(table, z(4), z(5), z(n), z(n), z(2), z(1))
        got = page_slots(lens, _i32(new, dev), table, free, ring, n, out=out)
        assert got.table is table
        _same(got, m.step(new, n, [False] * 4), free, m)
        lens, ring = got.lens, got.ring
    # in place, and rows that start anew
    out = PageSlots(table, *(torch.empty(n, dtype=torch.int32, device=dev) for n in (4, 5, 9, 9, 2, 1)))
    got = page_slots(lens, _i32([5, 1, 1, 2], dev), table, free, ring, 9, reset=torch.tensor([1, 0, 0, 1], dtype=torch.bool, device=dev), out=out)
    _same(got, m.step([5, 1, 1, 2], 9, [True, False, False, True]), free, m)


@pytest.mark.parametrize("lens,new,ring", [([-1, 2], [1, 1], [0, 5]), ([1, 129], [0, 0], [0, 5]), ([1, 2], [-1, 1], [0, 5]), ([1, 2], [1, 1], [5, 0]),
                                           ([1, 2], [1, 1], [-1, 2]), ([1, 2], [1, 1], [0, 6]), ([1, 2], [2**31 - 1, 2**31 - 1], [0, 5])])
def test_slots_impossible_counts(dev, lens, new, ring):
    table = _i32([[1, 0], [2, 0]], dev)
    free = _i32([3, 4, 5, 0, 0], dev)
    got = page_slots(_i32(lens, dev), _i32(new, dev), table, free, _i32(ring, dev), 8)
    assert got.status.item() & (8 | 2) and got.table.tolist() == table.tolist() and got.lens.tolist() == lens
    assert got.slots.tolist() == [-1] * 8 and got.ring.tolist() == ring and free.tolist() == [3, 4, 5, 0, 0]


def test_slots_refusals(dev):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    ok = dict(lens=z(2), new=z(2), table=z(2, 3), free=z(5), ring=z(2), n_tokens=4)
    page_slots(**ok)
    for name, bad in (("lens", z(3)), ("lens", z(2).long()), ("new", z(2, 1)), ("table", z(6)), ("table", z(3, 2).t()), ("ring", z(3)),
                      ("n_tokens", -1), ("reset", z(2)), ("reset", z(3).bool()), ("free", z(0))):
        with pytest.raises(ValueError):
            page_slots(**{**ok, name: bad})
    with pytest.raises(ValueError):
        page_slots(z(4097), z(4097), z(4097, 1), z(5), z(2), 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        page_slots(**{**ok, "lens": ok["lens"].cpu()})
    r = page_slots(**ok)
    with pytest.raises(ValueError, match="other memory"):
        page_slots(**ok, out=PageSlots(r.table, ok["lens"], r.starts, r.slots, r.positions, r.ring, r.status))
    with pytest.raises(ValueError, match="out.slots"):
        page_slots(**ok, out=PageSlots(r.table, r.lens, r.starts, z(3), r.positions, r.ring, r.status))


# ------------------------------------------------------------------ rope_axes
def _rotated(x, positions, scheme, inverse=False):
    """x [..., S, D] in 64 bits; positions [axes, ..., S] broadcast over x's leading dims."""
    inv = scheme.inv_freq().double().to(x.device)
    if isinstance(scheme, NoRope):
        return x.double()
    if isinstance(scheme, LinearScaled):
        inv = inv / scheme.factor
    axis = torch.tensor(scheme.freq_axes(), device=x.device)
    p = positions.double().to(x.device)
    p = p.expand(max(scheme.n_axes, 1), *p.shape[1:]) if p.shape[0] == 1 else p
    angle = p[axis].movedim(0, -1) * inv
    if inverse:
        angle = -angle
    h = inv.numel()
    a, b, rest = x[..., :h].double(), x[..., h : 2 * h].double(), x[..., 2 * h :].double()
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), rest], dim=-1)


def _rope_close(got, want, x, half):
    """One rounding to the type, on products of factors that are 2^-22 off at most (the sine and cosine 1.3e-7)
    and three fp32 roundings: each error is relative to the pair's two values."""
    eps = torch.finfo(got.dtype).eps
    xa = x.double().abs()
    pair = torch.cat([xa[..., :half] + xa[..., half : 2 * half]] * 2 + [0 * xa[..., 2 * half :]], dim=-1)
    tol = eps / 2 * want.abs() + (2.0**-22 + 3 * 2.0**-24) * (1 + eps) * pair + torch.finfo(got.dtype).tiny
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


SCHEMES = {
    "vanilla128": (Vanilla(theta=1e6, head_dim=128), 128),
    "vanilla64": (Vanilla(theta=10000.0, head_dim=64), 64),
    "vanilla256": (Vanilla(theta=10000.0, head_dim=256), 256),
    "vanilla80": (Vanilla(theta=10000.0, head_dim=80), 80),
    "vanilla24": (Vanilla(theta=10000.0, head_dim=24), 24),
    "vanilla6": (Vanilla(theta=10000.0, head_dim=6), 6),
    "linear": (LinearScaled(theta=10000.0, head_dim=64, factor=3.0), 64),
    "llama3": (Llama3(theta=5e5, head_dim=128, factor=8.0), 128),
    "yarn": (Yarn(theta=1e6, head_dim=128, factor=4.0, original_max_position_embeddings=4096), 128),
    "proportional": (Proportional(theta=1e6, head_dim=256, partial_rotary_factor=0.25), 256),
    "axes": (MRope(theta=1e6, head_dim=128, mrope_section=[16, 24, 24]), 128),
    "axes_partial": (MRope(theta=1e7, head_dim=256, partial_rotary_factor=0.25, mrope_section=[11, 11, 10], interleaved=True), 256),
    "axes_interleaved": (MRope(theta=1e6, head_dim=128, mrope_section=[24, 20, 20], interleaved=True), 128),
    "axes_two": (MRope(theta=1e4, head_dim=64, mrope_section=[20, 12]), 64),
    "partial_odd": (MRope(theta=1e4, head_dim=128, partial_rotary_factor=0.28125), 128),
    "norope": (NoRope(head_dim=64), 64),
}


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("name", list(SCHEMES))
def test_rope_axes(dev, name, dtype):
    scheme, D = SCHEMES[name]
    half = 0 if name == "norope" else len(scheme.freq_axes())
    g = torch.Generator(device=dev).manual_seed(len(name))
    for B, S, Hq, Hkv in ((1, 1, 4, 2), (2, 37, 3, 1), (3, 130, 1, 5)):
        # as projections leave them, and a slice of a larger tensor
        q = torch.randn(B, S, Hq, D, generator=g, device=dev).to(dtype).transpose(1, 2)
        k = torch.randn(B, Hkv + 1, S + 3, D, generator=g, device=dev).to(dtype)[:, 1:, 3:]
        for axes in {1, scheme.n_axes}:
            pos = torch.randint(0, 100000, (axes, B, S), generator=g, device=dev)
            qo, ko = rope_axes(q, k, pos, scheme)
            assert qo.is_contiguous() and ko.is_contiguous()
            _rope_close(qo, _rotated(q, pos[:, :, None], scheme), q, half)
            _rope_close(ko, _rotated(k, pos[:, :, None], scheme), k, half)
            qi, none = rope_axes(qo, None, pos.int(), scheme, inverse=True)
            assert none is None
            _rope_close(qi, _rotated(qo, pos[:, :, None], scheme, inverse=True), qo, half)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rope_far_positions(dev, dtype):
    """Angles stay exact where position * frequency in 32 bits has lost them."""
    scheme = Vanilla(theta=1e6, head_dim=128)
    pos = torch.tensor([0, 1, -1, -70000, 2**24 + 1, 10**8 + 7, 2**31 - 1], device=dev)
    x = torch.randn(1, 2, 7, 128, device=dev).to(dtype)
    got, _ = rope_axes(x, None, pos, scheme)
    # the angles in exact arithmetic on the host
    from fractions import Fraction

    pi = Fraction("3.14159265358979323846264338327950288419716939937511")
    turn = [[float(Fraction(p) * Fraction(f) / (2 * pi) % 1) for f in scheme.inv_freq().tolist()] for p in pos.tolist()]
    angle = torch.tensor(turn, dtype=torch.float64, device=dev) * 2 * math.pi
    a, b = x[..., :64].double(), x[..., 64:].double()
    _rope_close(got, torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1), x, 64)


def test_rope_positions_forms_and_in_place(dev):
    scheme = MRope(theta=1e6, head_dim=64, mrope_section=[8, 12, 12])
    q, k = torch.randn(2, 4, 9, 64, device=dev).half(), torch.randn(2, 2, 9, 64, device=dev).half()
    pos = torch.randint(0, 5000, (3, 2, 9), device=dev)
    full = rope_axes(q, k, pos, scheme)
    wide = torch.zeros(3, 2, 18, dtype=torch.int32, device=dev)
    wide[:, :, ::2] = pos.int()
    for a, b in zip(rope_axes(q, k, wide[:, :, ::2], scheme), full):  # strided, 32 bits
        assert torch.equal(a, b)
    one = pos[:, :1].contiguous()
    for p, e in ((one, one.expand(3, 2, 9)), (one[0], one[:1].expand(3, 2, 9)), (one[0, 0], one[:1].expand(3, 2, 9)), (pos[:1], pos[:1].expand(3, 2, 9))):
        for a, b in zip(rope_axes(q, k, p, scheme), rope_axes(q, k, e.contiguous(), scheme)):
            assert torch.equal(a, b)
    q2, k2 = q.clone(), k.clone()
    assert rope_axes(q2, k2, pos, scheme, out=(q2, k2))[0] is q2
    assert torch.equal(q2, full[0]) and torch.equal(k2, full[1])
    # rows that are not 16-byte aligned, and another memory order of the result
    buf = torch.randn(2, 4, 9, 65, device=dev).half()
    buf[..., 1:] = q
    dst = torch.zeros(2, 9, 4, 64, device=dev).half().transpose(1, 2)
    a, _ = rope_axes(buf[..., 1:], None, pos, scheme, out=(dst, None))
    assert a is dst and torch.equal(a, full[0])
    assert rope_axes(q[:, :, :0], None, pos[:, :, :0], scheme)[0].shape == (2, 4, 0, 64)


def test_rope_refusals(dev):
    s = Vanilla(theta=1e6, head_dim=64)
    q, p = torch.randn(1, 2, 5, 64, device=dev).half(), torch.arange(5, device=dev)
    rope_axes(q, None, p, s)
    for args in ((None, None, p, s), (q[0], None, p, s), (q.double(), None, p, s), (q, q.bfloat16(), p, s), (q, q[:, :, :3], p, s),
                 (q, None, p.float(), s), (q, None, p[:4], s), (q, None, p.expand(3, 5), s), (q, None, p.expand(3, 1, 5), s),
                 (q[..., :32], None, p, s), (q, None, p, MRope(theta=1e6, head_dim=64, mrope_section=[8, 8])),
                 (q, None, p, MRope(theta=1e6, head_dim=64, mrope_section=[8, 12, 12], interleaved=True))):
        with pytest.raises(ValueError):
            rope_axes(*args)
    with pytest.raises(ValueError):
        rope_axes(q, None, p, s, out=(q.float(), None))
    w = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        rope_axes(w, None, p, s)
    with torch.no_grad():
        rope_axes(w, None, p, s)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rope_axes(q.cpu(), None, p, s)


# --------------------------------------------------------------- paged_append
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name,Hq,Hkv", [("vanilla128", 8, 2), ("vanilla64", 14, 2), ("vanilla24", 3, 3), ("axes", 7, 1), ("axes_partial", 2, 2), (None, 0, 3)])
def test_append(dev, name, Hq, Hkv, dtype):
    scheme, D = SCHEMES[name] if name else (None, 72)
    g = torch.Generator(device=dev).manual_seed(Hq + 17)
    for T in (1, 5, 300):
        pool = TokenPagePool(T + 3, Hkv, D, dtype, dev)
        pool.k.normal_(generator=g)
        pool.v.normal_(generator=g)
        qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=dev).to(dtype)
        q, k, v = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv], qkv[:, Hq + Hkv :]
        slots = (torch.randperm((T + 3) * PAGE_TOKENS, generator=g, device=dev)[:T] + PAGE_TOKENS).int()
        if T > 1:  # no place, the page without tokens, past the pages
            slots[0], slots[1], slots[2], slots[4] = -1, 63, (T + 4) * PAGE_TOKENS, 2**31 - 1
        pos = torch.randint(0, 50000, (scheme.n_axes, T), generator=g, device=dev) if scheme else None
        kw, vw = pool.k.double(), pool.v.double()
        for t, s in enumerate(slots.tolist()):
            if PAGE_TOKENS <= s < (T + 4) * PAGE_TOKENS:
                kw[s // PAGE_TOKENS, :, s % PAGE_TOKENS] = _rotated(k[t, :, None], pos[:, t, None, None], scheme)[:, 0] if scheme else k[t].double()
                vw[s // PAGE_TOKENS, :, s % PAGE_TOKENS] = v[t].double()
        half = len(scheme.freq_axes()) if scheme else 0
        kx = pool.k.clone()
        live = [(t, s) for t, s in enumerate(slots.tolist()) if PAGE_TOKENS <= s < (T + 4) * PAGE_TOKENS]
        for t, s in live:
            kx[s // PAGE_TOKENS, :, s % PAGE_TOKENS] = k[t]
        version = pool.k._version
        qo = paged_append(k, v, pool.k, pool.v, slots, q=q if Hq else None, positions=pos, scheme=scheme)
        assert pool.k._version > version
        assert torch.equal(pool.v.double(), vw)
        _rope_close(pool.k, kw, kx, half)
        if Hq:
            _rope_close(qo, _rotated(q.transpose(0, 1), pos[:, None], scheme).transpose(0, 1), q, half)
            # the same values as the rotation alone
            both = rope_axes(q.transpose(0, 1)[None], k.transpose(0, 1)[None], pos[:, None], scheme)
            assert torch.equal(both[0][0].transpose(0, 1), qo)
            for t, s in live:
                assert torch.equal(pool.k[s // PAGE_TOKENS, :, s % PAGE_TOKENS], both[1][0, :, t])


def test_append_refusals(dev):
    pool = TokenPagePool(4, 2, 64, F16, dev)
    k, s = torch.randn(5, 2, 64, device=dev).half(), torch.arange(64, 69, device=dev).int()
    sch, p = Vanilla(theta=1e4, head_dim=64), torch.arange(5, device=dev)
    paged_append(k, k, pool.k, pool.v, s)
    ok = dict(k=k, v=k, k_pages=pool.k, v_pages=pool.v, slots=s)
    for bad in (dict(v=k[:3]), dict(k=k.float()), dict(v=k.bfloat16()), dict(k=k[:, :1], v=k[:, :1]), dict(slots=s.long()), dict(slots=s[:3]),
                dict(k_pages=pool.k.bfloat16()), dict(v_pages=pool.v[:2]), dict(k_pages=pool.k[:, :, :32], v_pages=pool.v[:, :, :32]),
                dict(k_pages=pool.k.transpose(0, 1), v_pages=pool.v.transpose(0, 1)), dict(scheme=sch), dict(positions=p), dict(q=k),
                dict(scheme=sch, positions=p[:3]), dict(scheme=sch, positions=p.float()), dict(scheme=sch, positions=p, q=k[:3]),
                dict(scheme=Vanilla(theta=1e4, head_dim=128), positions=p), dict(scheme=sch, positions=p.expand(3, 5)),
                dict(k=k.clone().requires_grad_()), dict(scheme=sch, positions=p, q=k, q_out=k[:3])):
        with pytest.raises(ValueError):
            paged_append(**{**ok, **bad})


# ------------------------------------------------------------ paged_attention
def _pages(gen, dev, lens, Hkv, D, dtype, extra=3, junk=None, chan=True):
    """A shuffled pool for rows of these lengths; `junk` stands in every place that holds no token."""
    counts = [-(-n // PAGE_TOKENS) for n in lens]
    total = sum(counts) + extra
    ids = (torch.randperm(total, generator=gen, device=dev) + 1).tolist()
    table = torch.zeros(len(lens), max(max(counts), 1) + 1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = torch.tensor(ids[at : at + c], dtype=torch.int32)
        at += c
    scale = torch.exp(0.5 * torch.randn(1, Hkv, 1, D, generator=gen, device=dev)) if chan else 1.0
    k = (torch.randn(total + 1, Hkv, PAGE_TOKENS, D, generator=gen, device=dev) * scale).to(dtype)
    v = torch.randn(total + 1, Hkv, PAGE_TOKENS, D, generator=gen, device=dev).to(dtype)
    if junk is not None:
        used = torch.zeros(total + 1, PAGE_TOKENS, dtype=torch.bool, device=dev)
        for b, n in enumerate(lens):
            for j in range(counts[b]):
                used[table[b, j], : min(PAGE_TOKENS, n - j * PAGE_TOKENS)] = True
        for x in (k, v):
            x.masked_fill_(~used[:, None, :, None], junk)
    return k, v, table.to(dev)


def _reference(q, k_pages, v_pages, table, lens, starts, scale, mask):
    """(output, tolerance) in 64 bits: a rounding of the output, of each probability and of the scores' fp32 sums."""
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
        seen = torch.ones(n, L, dtype=torch.bool, device=q.device)
        if mask == "bottom_right":
            seen = seen.tril(L - n)
        for h in range(Hkv):
            k, v = (x[ids, h].double().reshape(-1, D)[:L] for x in (k_pages, v_pages))
            qh = q[s:e, h * G : (h + 1) * G].double().transpose(0, 1).reshape(G * n, D)
            vis = seen.repeat(G, 1)
            x = (qh @ k.t()) * scale
            p = torch.softmax(x.masked_fill(~vis, -math.inf), dim=-1).nan_to_num(0.0)
            o = p @ v
            # a score's fp32 sum: D products, each addition 2^-24 of the sum of their sizes (and the scale, the
            # difference to the maximum, the exponential: a few more); the maximum's own error cancels
            ds = ((D + 8) * 2.0**-24 * scale * (qh.abs() @ k.abs().t())).masked_fill(~vis, 0.0).amax(-1, keepdim=True)
            spread = p @ v.abs()
            # fp16 probabilities under 2^-14 of the maximum's lose up to 2^-25 each, absolutely
            small = (2.0**-25 * vis.sum(-1, keepdim=True) * v.abs().amax() / p.amax(-1, keepdim=True).clamp(min=1e-30).reciprocal()
                     if q.dtype == F16 else 0.0)
            t = u * o.abs() + (2 * u + 2 * ds) * (1 + u) * spread + small + torch.finfo(q.dtype).tiny
            out[s:e, h * G : (h + 1) * G] = o.reshape(G, n, D).transpose(0, 1)
            tol[s:e, h * G : (h + 1) * G] = t.reshape(G, n, D).transpose(0, 1)
    return out, tol


def _check(got, want, tol, what=""):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{what}: {float((err / tol.clamp(min=1e-300)).nan_to_num(math.inf).max())} of the tolerance"


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


ROWS = {
    "one": ([1], [1]),
    "step": ([1, 2, 63, 64, 65, 128, 700], [1] * 7),
    "step_long": ([5000, 3], [1, 1]),
    "spec": ([70, 5, 1300], [4, 5, 3]),
    "chunk": ([300], [300]),
    "chunks": ([64, 500, 129, 1, 1000], [64, 37, 129, 1, 250]),
    "mixed": ([2000, 900, 31, 65], [1, 333, 31, 1]),
    "empty": ([0, 40, 10, 0, 200], [0, 0, 4, 0, 3]),
    "none_visible": ([0, 3, 70], [2, 9, 71]),
    "many": ([(37 * i) % 150 for i in range(70)], [min((37 * i) % 150, i % 3) for i in range(70)]),
}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", list(ROWS))
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (14, 2, 64), (16, 8, 256), (3, 3, 128), (20, 1, 64), (6, 2, 80), (4, 4, 8), (2, 1, 200), (5, 1, 40)])
def test_attention(dev, Hq, Hkv, D, rows, dtype):
    lens, new = ROWS[rows]
    g = torch.Generator(device=dev).manual_seed(D + len(rows))
    # what stands where no token does must not count
    k, v, table = _pages(g, dev, lens, Hkv, D, dtype, junk=math.nan)
    q = torch.randn(sum(new), Hq, D, generator=g, device=dev).to(dtype)
    starts = _starts(new)
    for mask in ("bottom_right", "none"):
        want, tol = _reference(q, k, v, table, lens, starts, 1 / math.sqrt(D), mask)
        got = paged_attention(q, k, v, table, _i32(lens, dev), _i32(starts, dev), mask=mask)
        _check(got, want, tol, mask)
        again = paged_attention(q, k, v, table, _i32(lens, dev), _i32(starts, dev), mask=mask)
        assert torch.equal(got, again)


@pytest.mark.parametrize("new", [1, 3, 100])
def test_attention_strides_tail_and_scale(dev, new):
    g = torch.Generator(device=dev).manual_seed(new)
    lens, Hq, Hkv, D = [500, 1200, 64], 12, 4, 128
    starts = _starts([new] * 3)
    k, v, table = _pages(g, dev, lens, Hkv, D, F16)
    T = starts[-1] + 9
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=dev).half()
    q = qkv[:, :Hq]
    args = (q, k, v, table, _i32(lens, dev), _i32(starts, dev))
    want, tol = _reference(q, k, v, table, lens, starts, 0.3, "bottom_right")
    got = paged_attention(*args, sm_scale=0.3)
    _check(got, want, tol)
    assert not got[starts[-1] :].any()  # a new tensor: zeros behind the last sequence
    out = torch.full((Hq, T, D + 8), 7.0, device=dev).half()[:, :, 4 : 4 + D].transpose(0, 1)
    got2 = paged_attention(*args, sm_scale=0.3, out=out)
    assert got2 is out and torch.equal(out[: starts[-1]], got[: starts[-1]])
    assert bool((out[starts[-1] :] == 7.0).all())  # the caller's: left as they were


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (6, 3, 64)])
def test_attention_into_its_queries(dev, Hq, Hkv, D):
    """out = q, with tiles of both kernels, cut and whole, and one that is walked again; strides of one-element axes."""
    lens, new = [2500, 300, 1, 40, 900], [1, 300, 1, 3, 130]
    g = torch.Generator(device=dev).manual_seed(Hq)
    k, v, table = _pages(g, dev, lens, Hkv, D, BF16)
    v[table[4, 13], :, 60] = math.inf
    starts = _starts(new)
    q = torch.randn(starts[-1] + 2, Hq, D, generator=g, device=dev).to(BF16)
    args = (k, v, table, _i32(lens, dev), _i32(starts, dev))
    want, rest = paged_attention(q, *args), q[starts[-1] :].clone()
    got = paged_attention(q, *args, out=q)
    assert got is q
    a, b = got[: starts[-1]], want[: starts[-1]]
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num()) and torch.equal(got[starts[-1] :], rest)
    x = torch.randn(Hq, D, generator=g, device=dev).to(BF16)
    one = x.as_strided((1, Hq, D), (3, D, 1))
    assert torch.equal(paged_attention(one, k, v, table[:1], _i32([70], dev), _i32([0, 1], dev)),
                       paged_attention(x[None], k, v, table[:1], _i32([70], dev), _i32([0, 1], dev)))
    with pytest.raises(ValueError, match="out must be"):
        paged_attention(q, *args, out=q[:1].expand(starts[-1] + 2, Hq, D))


def test_attention_extreme_scores(dev):
    """Scores of thousands, equal keys, infinite keys: as a softmax in 64 bits has them."""
    lens, new, H, D = [130, 70, 65], [1, 2, 65], 2, 64
    starts = _starts(new)
    k = torch.randn(8, H, PAGE_TOKENS, D, device=dev).bfloat16()
    v = torch.randn(8, H, PAGE_TOKENS, D, device=dev).bfloat16()
    table = _i32([[1, 2, 3], [4, 5, 0], [6, 7, 0]], dev)
    q = torch.randn(starts[-1], H, D, device=dev).bfloat16()
    lt, st = _i32(lens, dev), _i32(starts, dev)
    for scale in (100.0, 1e-3):
        want, tol = _reference(q, k, v, table, lens, starts, scale, "bottom_right")
        _check(paged_attention(q, k, v, table, lt, st, sm_scale=scale), want, tol, str(scale))
    k[:] = 0.5  # equal scores: the mean of the visible values
    want, tol = _reference(q, k, v, table, lens, starts, 1.0, "bottom_right")
    _check(paged_attention(q, k, v, table, lt, st, sm_scale=1.0), want, tol)
    # a key whose scores are -inf has no weight, one with +inf or NaN makes the queries that see it NaN
    q = q.abs() + 1
    k[2, :, 10] = -math.inf  # row 0's key 74
    k[5, :, 3] = math.inf    # row 1's key 67: seen by both of its queries (68 and 69)
    k[7, :, 0] = math.nan    # row 2's key 64: seen by its last query alone
    got = paged_attention(q, k, v, table, lt, st, sm_scale=1.0)
    keep = torch.arange(130, device=dev) != 74
    vv = torch.cat([v[1], v[2], v[3]], dim=1)[:, :130].double()
    assert bool(((got[0].double() - vv[:, keep].mean(1)).abs() <= 2.0**-6).all())
    assert bool(got[1:3].isnan().all()) and bool(got[-1].isnan().all()) and not bool(got[3:-1].isnan().any())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (3, 3, 64), (4, 2, 256), (2, 1, 80)])
@pytest.mark.parametrize("lens,new", [([70, 33, 200], [3, 4, 2]), ([64, 300], [64, 170]), ([130, 1, 700], [130, 1, 97])])
def test_attention_values_that_are_no_numbers(dev, lens, new, Hq, Hkv, D, dtype):
    """An infinity or a NaN in V reaches the queries that see its key, and no other."""
    g = torch.Generator(device=dev).manual_seed(D)
    k, v, table = _pages(g, dev, lens, Hkv, D, dtype, junk=math.nan)
    q = torch.randn(sum(new), Hq, D, generator=g, device=dev).to(dtype)
    starts = _starts(new)
    args = (table, _i32(lens, dev), _i32(starts, dev))
    odd = v.clone()
    up, down = torch.zeros(2, len(lens), max(lens), Hkv, D, dtype=torch.bool, device=dev)
    for b, (L, n) in enumerate(zip(lens, new)):
        # the last token, one among the new ones, the last one before them
        for j, (t, x) in enumerate(zip((L - 1, L - 1 - n // 2, max(L - n - 1, 0)), (math.nan, math.inf, -math.inf))):
            at = (table[b, t // PAGE_TOKENS], (b + j) % Hkv, t % PAGE_TOKENS)
            odd[(*at, slice(j, D, 5))] = x
            v[(*at, slice(j, D, 5))] = 0.0
            up[b, t, (b + j) % Hkv, j::5] |= not x < 0
            down[b, t, (b + j) % Hkv, j::5] |= not x > 0
    want = paged_attention(q, k, v, *args)
    got = paged_attention(q, k, odd, *args)
    for b, (L, n) in enumerate(zip(lens, new)):
        for i in range(n):
            for kind, sign in ((up, math.inf), (down, -math.inf)):
                hit = kind[b, : L - n + i + 1].any(0).repeat_interleave(Hq // Hkv, 0)
                want[starts[b] + i] = torch.where(hit, want[starts[b] + i] + sign, want[starts[b] + i])
    wrong = ~((got == want) | (got.isnan() & want.isnan()))
    at = wrong.nonzero()[:4].tolist()
    assert not at, [(i, float(got[tuple(i)]), float(want[tuple(i)])) for i in at]


def test_attention_device_data_out_of_range(dev):
    """Lengths past the table, page ids outside the pool, starts past q: kept inside the tensors."""
    H, D = 2, 64
    k = torch.randn(4, H, PAGE_TOKENS, D, device=dev).half()
    v = torch.randn(4, H, PAGE_TOKENS, D, device=dev).half()
    q = torch.randn(3, H, D, device=dev).half()
    ok = paged_attention(q, k, v, _i32([[1, 2], [3, 0], [1, 0]], dev), _i32([128, 64, 5], dev), _i32([0, 1, 2, 3], dev))
    got = paged_attention(q, k, v, _i32([[1, 2], [3, 0], [1, 0]], dev), _i32([2**31 - 1, 64, 5], dev), _i32([-4, 1, 2, 99], dev))
    assert torch.equal(ok, got)
    a = paged_attention(q, k, v, _i32([[-5, 2], [3, 0], [99, 0]], dev), _i32([128, 64, 5], dev), _i32([0, 1, 2, 3], dev))
    b = paged_attention(q, k, v, _i32([[0, 2], [3, 0], [0, 0]], dev), _i32([128, 64, 5], dev), _i32([0, 1, 2, 3], dev))
    assert torch.equal(a, b)
    neg = paged_attention(q, k, v, _i32([[1, 2], [3, 0], [1, 0]], dev), _i32([-3, 64, 5], dev), _i32([0, 1, 2, 3], dev))
    assert not neg[0].any() and torch.equal(neg[1:], ok[1:])


def test_attention_streams_graph_and_two_plans(dev):
    g = torch.Generator(device=dev).manual_seed(5)
    lens, H, D = [3000, 200, 1500], 4, 128
    k, v, table = _pages(g, dev, [4000, 300, 1600], H, D, F16)
    lt, st = _i32(lens, dev), _i32([0, 1, 2, 3], dev)
    q = torch.randn(3, 4 * H, D, generator=g, device=dev).half()
    q2 = torch.randn(3, 4 * H, D, generator=g, device=dev).half()
    plan, other = PagedAttentionPlan(q, k, v, table, lt, st), PagedAttentionPlan(q2, k, v, table, lt, st)
    assert plan.workspace is not None
    want, want2 = plan.run().clone(), other.run().clone()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    for _ in range(5):  # the two at once
        with torch.cuda.stream(side):
            other.run()
        plan.run()
    torch.cuda.synchronize()
    assert torch.equal(plan.out, want) and torch.equal(other.out, want2)
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
    with torch.cuda.graph(graph2):
        other.run()
    for i in range(4):
        lt.copy_(_i32([3000 + i, 200 + 9 * i, 1500 - 400 * i], dev))
        plan.out.zero_()
        other.out.zero_()
        graph.replay()
        graph2.replay()
        a, b = plan.out.clone(), other.out.clone()
        torch.cuda.synchronize()
        assert torch.equal(a, paged_attention(q, k, v, table, lt, st)) and torch.equal(b, paged_attention(q2, k, v, table, lt, st)), i


def test_attention_refusals(dev):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    h = lambda *s: torch.zeros(s, dtype=F16, device=dev)  # noqa: E731
    ok = dict(q=h(3, 4, 64), k_pages=h(5, 2, 64, 64), v_pages=h(5, 2, 64, 64), table=z(2, 3), lens=z(2), starts=z(3))
    paged_attention(**ok)
    for bad in (dict(q=h(3, 4, 32)), dict(q=h(3, 3, 64)), dict(q=h(1, 3, 4, 64)), dict(q=ok["q"].float()), dict(q=ok["q"].bfloat16()),
                dict(k_pages=h(5, 2, 32, 64)), dict(v_pages=h(4, 2, 64, 64)), dict(k_pages=h(5, 2, 64, 12), v_pages=h(5, 2, 64, 12), q=h(3, 4, 12)),
                dict(k_pages=h(5, 2, 64, 264), v_pages=h(5, 2, 64, 264), q=h(3, 4, 264)), dict(table=z(2, 3).long()), dict(table=z(6)),
                dict(lens=z(3)), dict(starts=z(2)), dict(mask="top_left"), dict(sm_scale=0.0), dict(sm_scale=-1.0), dict(sm_scale=math.nan),
                dict(sm_scale=math.inf), dict(out=h(3, 4, 32)), dict(out=ok["q"].float()), dict(q=h(3, 4, 65)[..., 1:]),
                dict(q=ok["q"].clone().requires_grad_())):
        with pytest.raises(ValueError):
            paged_attention(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_attention(**{**ok, "lens": ok["lens"].cpu()})
    assert paged_attention(**{**ok, "q": h(0, 4, 64)}).shape == (0, 4, 64)


# ------------------------------------------------------------ a serving step
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_serving_steps(dev, dtype):
    """Prompts in chunks of different lengths, decoding, a row that is replaced: slots, append and
    attention together, against each row's own tokens in 64 bits; then the rows are compressed."""
    B, Hq, Hkv, D = 3, 8, 2, 128
    scheme = MRope(theta=1e6, head_dim=D, mrope_section=[16, 24, 24])
    pool = TokenPagePool(60, Hkv, D, dtype, dev)
    pool.k.fill_(math.nan)
    pool.v.fill_(math.nan)
    state = pool.start(B, 20)
    rows = [[torch.zeros(0, Hkv, D, dtype=torch.float64, device=dev) for _ in range(2)] for _ in range(B)]
    g = torch.Generator(device=dev).manual_seed(3)
    for step, (new, reset) in enumerate((([200, 0, 65], None), ([100, 1, 1], None), ([1, 130, 1], None), ([1, 1, 1], None), ([70, 1, 1], [1, 0, 0]), ([1, 0, 1], None))):
        T = sum(new) + 4
        rs = None if reset is None else torch.tensor(reset, dtype=torch.bool, device=dev)
        state = pool.step(state, _i32(new, dev), T, reset=rs).check()
        qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=dev).to(dtype)
        q, k, v = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv], qkv[:, Hq + Hkv :]
        pos = torch.stack([state.positions.long(), state.positions.long() // 3, state.positions.long() % 7])
        qr = paged_append(k, v, pool.k, pool.v, state.slots, q=q, positions=pos, scheme=scheme)
        out = paged_attention(qr, pool.k, pool.v, state.table, state.lens, state.starts)
        kr = rope_axes(None, k.transpose(0, 1)[None], pos[:, None], scheme)[1][0].transpose(0, 1)
        starts = _starts(new)
        for b in range(B):
            if reset and reset[b]:
                rows[b] = [x[:0] for x in rows[b]]
            at = slice(starts[b], starts[b + 1])
            rows[b] = [torch.cat([x, y[at].double()]) for x, y in zip(rows[b], (kr, v))]
            n, L = new[b], rows[b][0].shape[0]
            if n == 0:
                continue
            kk, vv = (x.repeat_interleave(Hq // Hkv, 1).transpose(0, 1) for x in rows[b])
            x = qr[at].double().transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(D)
            x = x.masked_fill(~torch.ones(n, L, dtype=torch.bool, device=dev).tril(L - n), -math.inf)
            want = (torch.softmax(x, -1) @ vv).transpose(0, 1)
            # (values of a few units: the roundings of the output and of the probabilities)
            assert float((out[at].double() - want).abs().max()) <= 3 * torch.finfo(dtype).eps / 2 * float(vv.abs().max()), (step, b)
        assert not out[starts[-1] :].any()
    lens = state.lens.tolist()
    assert lens == [71, 133, 70]
    # the rows' tokens as the compression takes them
    ks, vs = pool.gather(state.table, max(lens))
    for b, n in enumerate(lens):
        assert torch.equal(ks[b, :, :n].double(), rows[b][0].transpose(0, 1)) and torch.equal(vs[b, :, :n].double(), rows[b][1].transpose(0, 1))
    if dtype == F16:
        gone = torch.arange(max(lens), device=dev)[None, :] >= state.lens[:, None]
        for x in (ks, vs):
            x.masked_fill_(gone[:, None, :, None], 0.0)
        kq, sk = quant_k_int4(ks)
        vq, sv = quant_v_int4(vs)
        table, _ = MiddlePagePool(10, Hkv, D, dev).store(kq, vq, sv, lens)
        assert table.shape == (B, 3)


def test_attention_agrees_with_the_prefill(dev):
    """Rows of equal lengths: what the tiered prefill gives for the same keys."""
    B, Hq, Hkv, D, L, n = 2, 8, 2, 128, 700, 150
    g = torch.Generator(device=dev).manual_seed(9)
    k, v, table = _pages(g, dev, [L] * B, Hkv, D, F16)
    q = torch.randn(B, n, Hq, D, generator=g, device=dev).half()
    full = [x[table.long()].permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)[:, :, :L].contiguous() for x in (k, v)]
    ref = tiered_prefill_attention(q.transpose(1, 2), tuple(x[:, :, L - n :] for x in full), recent=tuple(x[:, :, : L - n] for x in full))
    got = paged_attention(q.reshape(B * n, Hq, D), k, v, table, _i32([L] * B, dev), _i32([0, n, 2 * n], dev)).reshape(B, n, Hq, D)
    bound = 4 * torch.finfo(F16).eps / 2 * float(v.abs().max())  # two outputs, a rounding of the probabilities and of the output each
    assert float((got.transpose(1, 2).double() - ref.double()).abs().max()) <= bound


def _step_inputs(g, dev, T, Hq, Hkv, D, dtype):
    return torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=dev).to(dtype)


def _step(pool, state, new, qkv, T, Hq, Hkv, scheme):
    state = pool.step(state, new, T)
    q, k, v = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv], qkv[:, Hq + Hkv :]
    qr = paged_append(k, v, pool.k, pool.v, state.slots, q=q, positions=state.positions, scheme=scheme)
    return state, paged_attention(qr, pool.k, pool.v, state.table, state.lens, state.starts)


def test_steps_in_two_graphs(dev):
    """A decoding step and one with a chunk, captured and replayed in turn over one pool, with eager steps of
    another pool between them: every replay as the eager step."""
    B, Hq, Hkv, D, dtype = 5, 8, 2, 64, BF16
    scheme = Llama3(theta=5e5, head_dim=D)
    eager, pool = (TokenPagePool(80, Hkv, D, dtype, dev) for _ in range(2))
    g = torch.Generator(device=dev).manual_seed(11)
    kinds = ([1] * B, [1, 150, 1, 0, 1])
    a = eager.start(B, 12)
    lens, table = (torch.zeros_like(x) for x in (a.lens, a.table))
    ring = pool.ring.clone()
    graphs = []
    for new in kinds:
        T = sum(new) + 3
        x = dict(new=_i32(new, dev), qkv=torch.zeros(T, Hq + 2 * Hkv, D, dtype=dtype, device=dev), T=T)

        def run(x=x):
            st = PageSlots(table, lens, None, None, None, ring, None)
            pool.ring = ring
            st, out = _step(pool, st, x["new"], x["qkv"], x["T"], Hq, Hkv, scheme)
            for dst, src in ((lens, st.lens), (table, st.table), (ring, st.ring)):
                dst.copy_(src)
            return st, out

        keep = [t.clone() for t in (lens, table, ring, pool.free, pool.k, pool.v)]
        run()
        for t, old in zip((lens, table, ring, pool.free, pool.k, pool.v), keep):
            t.copy_(old)
        x["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(x["graph"]):
            x["state"], x["out"] = run()
        graphs.append(x)
    for i in range(7):
        x = graphs[i % 2]
        qkv = _step_inputs(g, dev, x["T"], Hq, Hkv, D, dtype)
        a, want = _step(eager, a, x["new"], qkv, x["T"], Hq, Hkv, scheme)
        a.check()
        x["qkv"].copy_(qkv)
        x["graph"].replay()
        assert int(x["state"].status) == 0 and torch.equal(x["out"], want), i
        assert torch.equal(lens, a.lens) and torch.equal(table, a.table) and torch.equal(ring, a.ring)
        torch.cuda.synchronize()


def test_steps_on_another_stream(dev):
    """A step on a side stream while the default stream works on another pool's."""
    B, Hq, Hkv, D, dtype = 3, 4, 4, 128, F16
    scheme = Vanilla(theta=1e4, head_dim=D)
    g = torch.Generator(device=dev).manual_seed(12)
    new = _i32([300, 1, 64], dev)
    pools = [TokenPagePool(40, Hkv, D, dtype, dev) for _ in range(4)]
    xs = [_step_inputs(g, dev, 365, Hq, Hkv, D, dtype) for _ in range(4)]
    want = [_step(TokenPagePool(40, Hkv, D, dtype, dev), pools[0].start(B, 8), new, x, 365, Hq, Hkv, scheme)[1] for x in xs]
    starts = [p.start(B, 8) for p in pools]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream(dev) for _ in range(2)]
    got = [None] * 4
    for i in range(4):
        with torch.cuda.stream(sides[i % 2] if i < 3 else torch.cuda.default_stream(dev)):
            got[i] = _step(pools[i], starts[i], new, xs[i], 365, Hq, Hkv, scheme)[1]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_frequencies_are_not_uploaded_during_capture(dev):
    scheme = Vanilla(theta=123457.0, head_dim=64)
    q, pos = torch.randn(1, 2, 5, 64, device=dev).half(), torch.arange(5, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        buf = q * 2
        with pytest.raises(RuntimeError, match="once before capturing"):
            rope_axes(q, None, pos, scheme)
    want = rope_axes(q, None, pos, scheme)[0].clone()
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        out = rope_axes(q, None, pos, scheme)[0]
    for _ in range(3):
        out.zero_()
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(buf, q * 2)


def test_off_the_current_device(dev, monkeypatch):
    """Every entry point makes its tensors' GPU the current one for its launch (seen on one GPU by its guard)."""
    B, Hq, Hkv, D = 2, 4, 2, 64
    scheme = Vanilla(theta=1e4, head_dim=D)
    g = torch.Generator(device=dev).manual_seed(13)
    x, new = _step_inputs(g, dev, 70, Hq, Hkv, D, F16), _i32([64, 6], dev)
    pools = [TokenPagePool(9, Hkv, D, F16, dev) for _ in range(2)]
    states = [p.start(B, 2) for p in pools]
    want = _step(pools[0], states[0], new, x, 70, Hq, Hkv, scheme)[1]
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
        got = _step(pools[1], states[1], new, x, 70, Hq, Hkv, scheme)[1]
    assert len(entered) == 3 and torch.equal(got, want)


def test_offsets_past_32_bits(dev):
    """Pages and rows whose offsets pass 2^32 elements."""
    Hq, Hkv, D = 4, 8, 128
    page = Hkv * PAGE_TOKENS * D
    n_pages = 2**32 // page + 6
    k_pages, v_pages = (torch.empty(n_pages, Hkv, PAGE_TOKENS, D, dtype=BF16, device=dev) for _ in range(2))
    lens, new = [130, 1], [130, 1]
    ids = [n_pages - 1, 2, n_pages - 4, 2**31 // page + 1]
    table = _i32([[ids[0], ids[1], ids[2]], [ids[3], 0, 0]], dev)
    slots = _i32([64 * ids[i // 64] + i % 64 for i in range(130)] + [64 * ids[3]], dev)
    g = torch.Generator(device=dev).manual_seed(17)
    k, v = (torch.randn(131, Hkv, D, generator=g, device=dev).to(BF16) for _ in range(2))
    paged_append(k, v, k_pages, v_pages, slots)
    assert torch.equal(k_pages[ids[0], :, :].transpose(0, 1), k[:64]) and torch.equal(v_pages[ids[3], :, 0], v[130])
    # queries whose tokens lie 2^32 elements apart, in the pages' memory
    spare = k_pages.view(-1)
    q = torch.randn(131, Hkv * Hq, D, generator=g, device=dev).to(BF16)
    starts = _i32([0, 130, 131], dev)
    want = paged_attention(q, k_pages, v_pages, table, _i32(lens, dev), starts)
    ref, tol = _reference(q, k_pages, v_pages, table, lens, [0, 130, 131], 1 / math.sqrt(D), "bottom_right")
    _check(want, ref, tol)
    far = spare[3 * page :].as_strided((1, 2, Hq, D), (0, 2**32, D, 1))
    far.copy_(q[:2, :Hq][None])
    got = paged_attention(far[0], k_pages[:3, :Hq].contiguous(), v_pages[:3, :Hq].contiguous(), _i32([[2], [2]], dev), _i32([64, 64], dev),
                          _i32([0, 1, 2], dev))
    near = paged_attention(q[:2, :Hq].contiguous(), k_pages[:3, :Hq].contiguous(), v_pages[:3, :Hq].contiguous(), _i32([[2], [2]], dev),
                           _i32([64, 64], dev), _i32([0, 1, 2], dev))
    assert torch.equal(got, near)
    scheme, pos = Vanilla(theta=1e4, head_dim=D), _i32([5, 6], dev)
    xs = far.transpose(1, 2)
    assert torch.equal(rope_axes(xs, None, pos, scheme)[0], rope_axes(xs.contiguous(), None, pos, scheme)[0])
