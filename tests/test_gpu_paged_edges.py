"""The paged attention where its numbers are hard, against softmaxes in 64 bits, and rotations that must
not depend on how their rows lie in memory; what the paged operators refuse."""

from __future__ import annotations

import math

import pytest
import torch
from torch.autograd import forward_ad

from fade_amd.kernels import paged_append, paged_attention
from fade_amd.pages import PAGE_TOKENS, PageSlots, TokenPagePool, page_slots
from fade_amd.rope import Llama3, MRope, Proportional, Vanilla, rerope_gather, rope_axes
from test_gpu_paged import BF16, F16, F32, _check, _i32, _pages, _reference, _starts

pytestmark = pytest.mark.gpu


def _rows(x, table, L):
    """[B, Hkv, L, D] in 64 bits of rows of one length."""
    B, (_, H, _, D) = table.shape[0], x.shape
    return x[table[:, : -(-L // PAGE_TOKENS)].long()].permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)[:, :, :L].double().contiguous()


@pytest.mark.parametrize("gap", [10, 16, 20, 24, 28])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,new", [(600, 1), (150, 40)])  # tiles of 16 and of 256 matrix rows, one or more to a workgroup
def test_attention_of_a_light_tail(dev, B, new, dtype, gap):
    """One key takes the weight and has no value (an attention sink): the output is what keys 2^gap times lighter add up to."""
    L, Hq, Hkv, D = 450, 4, 2, 64
    g = torch.Generator(device=dev).manual_seed(gap)
    k, v, table = _pages(g, dev, [L] * B, Hkv, D, dtype)
    k.zero_()
    k[..., 0] = torch.randint(0, 33, k.shape[:3], generator=g, device=dev).to(dtype) / 64  # scores of 0 to 2 in powers of two, exactly
    v.copy_((torch.rand(v.shape, generator=g, device=dev) + 0.5) * 256)
    first = table[:, 0].long()
    k[first, :, 0, 0] = (gap + 2) / 4
    v[first, :, 0] = 0.0
    q = torch.zeros(B * new, Hq, D, device=dev, dtype=dtype)
    q[..., 0] = 4.0
    scale = math.log(2.0)
    got = paged_attention(q, k, v, table, _i32([L] * B, dev), _i32(_starts([new] * B), dev), sm_scale=scale)
    x = (4.0 * _rows(k, table, L)[..., 0])[:, :, None].expand(B, Hkv, new, L)
    seen = torch.ones(new, L, dtype=torch.bool, device=dev).tril(L - new)
    p = torch.softmax((x * math.log(2.0)).masked_fill(~seen, -math.inf), -1)
    o = p @ _rows(v, table, L)  # [B, Hkv, new, D], alike for the heads of a group
    want = o.permute(0, 2, 1, 3).repeat_interleave(Hq // Hkv, 2).reshape(B * new, Hq, D)
    # A rounding of the output, and: exponents of up to 32 in fp32, products and differences rounded (2^-24 of 32 each, four of
    # them: 2^-17), sums of 450 terms in fp32 and the exponential (2^-17 together).  The few-row kernel's probabilities are a
    # head and a rest (2^-17 of them in bf16), the wide one's rounded once, and their sum with them (2 u).
    u, few = torch.finfo(dtype).eps / 2, new == 1
    tol = (u + 2.0**-15 + (0 if few else 2 * u)) * want.abs()
    if dtype == F16:  # what fp16 cannot hold of a probability, next to one of 1: 2^-25 of the factor that they are held with
        tol += L * 384 * (2.0**-40 if few else 2.0**-34)
    _check(got, want, tol, f"gap {gap}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scale", [1e3, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("lens,new", [([300, 1, 700], [1, 1, 1]), ([300, 64, 1000], [300, 33, 150]), ([2000], [700])])
def test_attention_of_far_scores(dev, lens, new, scale, dtype):
    """Whole scores times a large factor: the mean of the values whose scores are the largest."""
    Hq, Hkv, D = 6, 3, 64
    g = torch.Generator(device=dev).manual_seed(len(lens))
    k, v, table = _pages(g, dev, lens, Hkv, D, dtype)
    k.copy_(torch.randint(-4, 5, k.shape, generator=g, device=dev))
    starts = _starts(new)
    q = torch.randint(-4, 5, (starts[-1], Hq, D), generator=g, device=dev).to(dtype)
    for mask in ("bottom_right", "none"):
        got = paged_attention(q, k, v, table, _i32(lens, dev), _i32(starts, dev), sm_scale=scale, mask=mask)
        # (differences of at least 1 are at least 1443 powers of two: nothing is left of any other key in 64 bits)
        want, _ = _reference(q, k, v, table, lens, starts, scale, mask)
        # equal keys have equal probabilities, which their sum takes as they are: the sums' roundings and the output's
        tol = (torch.finfo(dtype).eps / 2 + 2.0**-17) * want.abs() + 2.0**-17 * float(v.abs().max())
        _check(got, want, tol, mask)


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("scale", [2.0**-106, 1.0])
def test_attention_of_far_negative_scores(dev, new, scale):
    """Products of -2^106 and less: a query's keys are seen however low they all score."""
    L, H, D = 500, 2, 64
    g = torch.Generator(device=dev).manual_seed(new)
    k, v, table = _pages(g, dev, [L], H, D, BF16)
    q = torch.zeros(new, H, D, device=dev, dtype=BF16)
    q[..., 0] = 2.0**53
    k.zero_()
    k[..., 0] = -(2.0**53) * torch.randint(1, 9, k.shape[:3], generator=g, device=dev).to(BF16)
    got = paged_attention(q, k, v, table, _i32([L], dev), _i32([0, new], dev), sm_scale=scale)
    want, _ = _reference(q, k, v, table, [L], [0, new], scale, "bottom_right")
    # exact products; exponents of 12 at most that count: the roundings of the output, of each probability and of their sum,
    # and 2^-17 for the exponents' and the sums' in fp32
    u = torch.finfo(BF16).eps / 2
    _check(got, want, (u + 2.0**-17) * want.abs() + (2 * u + 2.0**-17) * float(v.abs().max()))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("scheme", [Vanilla(theta=1e6, head_dim=128), MRope(theta=1e6, head_dim=128, partial_rotary_factor=0.25)])
def test_rotation_of_unaligned_rows(dev, scheme, dtype):
    """Bit for bit that of aligned rows, and the two halves of a row alike: one fp32 sum, rounded to the type."""
    B, H, S, D = 2, 16, 200, 128
    g = torch.Generator(device=dev).manual_seed(7)
    x = torch.randn(B, H, S, D, generator=g, device=dev).to(dtype)
    pos = torch.randint(0, 5000, (B, S), generator=g, device=dev)
    want, _ = rope_axes(x, None, pos, scheme)
    buf = torch.zeros(B, H, S, D + 1, device=dev, dtype=dtype)
    buf[..., 1:] = x
    assert torch.equal(rope_axes(buf[..., 1:], None, pos, scheme)[0], want)
    # (x, y) and (-y, x) turn into (a, b) and (-b, a)
    h = len(scheme.freq_axes())
    y = torch.cat([-x[..., h : 2 * h], x[..., :h], x[..., 2 * h :]], -1)
    other, _ = rope_axes(y, None, pos, scheme)
    assert torch.equal(other[..., h : 2 * h], want[..., :h]) and torch.equal(-other[..., :h], want[..., h : 2 * h])
    if dtype != F32:
        pool = TokenPagePool(-(-B * S // PAGE_TOKENS), H, D, dtype, dev)
        k = torch.zeros(B * S, H, D + 1, device=dev, dtype=dtype)[..., 1:]
        k.copy_(x.transpose(1, 2).reshape(B * S, H, D))
        paged_append(k, k, pool.k, pool.v, torch.arange(B * S, device=dev).int() + PAGE_TOKENS, positions=pos.reshape(-1), scheme=scheme)
        got = pool.k[1:].transpose(1, 2).reshape(-1, H, D)[: B * S]
        assert torch.equal(got.view(B, S, H, D).transpose(1, 2), want)


def test_forward_mode_is_refused(dev):
    """A tangent would be lost: the calls that would lose it raise, whichever tensor has it."""
    D = 64
    g = torch.Generator(device=dev).manual_seed(1)
    q, pages = (torch.randn(s, generator=g, device=dev).half() for s in ((5, 2, D), (3, 2, PAGE_TOKENS, D)))
    ints = (_i32([[1, 2]], dev), _i32([70], dev), _i32([0, 5], dev))
    scheme, pos = Vanilla(theta=1e4, head_dim=D), torch.arange(5, device=dev)
    slots = pos.int() + PAGE_TOKENS
    calls = [lambda x, p: paged_attention(x, p, p, *ints), lambda x, p: rope_axes(x[None], None, pos[:2], scheme),
             lambda x, p: paged_append(x, x, p, p.clone(), slots, q=x, positions=pos, scheme=scheme)]
    for call in calls:
        call(q, pages.clone())
        with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            call(forward_ad.make_dual(q, torch.ones_like(q)), pages.clone())
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        calls[0](q, forward_ad.make_dual(pages, torch.ones_like(pages)))


def test_outputs_of_repeated_rows_are_refused(dev):
    D, T = 64, 6
    g = torch.Generator(device=dev).manual_seed(2)
    q = torch.randn(T, 4, D, generator=g, device=dev).half()
    pages = torch.randn(3, 4, PAGE_TOKENS, D, generator=g, device=dev).half()
    scheme, pos = Vanilla(theta=1e4, head_dim=D), torch.arange(T, device=dev)
    room = torch.zeros(T * 4 * D + 8, device=dev).half()
    for out in (q[:1].expand(T, 4, D), q[:, :1].expand(T, 4, D), room.as_strided((T, 4, D), (2 * D, D, 1)), room.as_strided((T, 4, D), (4 * D, D - 4, 1))):
        with pytest.raises(ValueError, match="no row twice"):
            rope_axes(q.transpose(0, 1)[None], None, pos, scheme, out=(out.transpose(0, 1)[None], None))
        with pytest.raises(ValueError, match="no row twice"):
            paged_append(q, q, pages, pages.clone(), pos.int() + PAGE_TOKENS, q=q, positions=pos, scheme=scheme, q_out=out)
        with pytest.raises(ValueError, match="no row twice"):
            paged_attention(q, pages, pages, _i32([[1]], dev), _i32([T], dev), _i32([0, T], dev), out=out)
    assert not room.any()
    other = room[: T * 4 * D].view(4, T, D).transpose(0, 1)  # rows in another order are fine
    assert rope_axes(q.transpose(0, 1)[None], None, pos, scheme, out=(other.transpose(0, 1)[None], None))[0] is not None
    paged_append(q, q, pages, pages.clone(), pos.int() + PAGE_TOKENS, q=q, positions=pos, scheme=scheme, q_out=other)
    paged_attention(q, pages, pages, _i32([[1]], dev), _i32([T], dev), _i32([0, T], dev), out=other)


def test_outputs_over_inputs_are_refused(dev):
    """An output may be its own input, or lie between the inputs' rows, and nothing else of the call's memory."""
    D, T, H = 64, 6, 4
    g = torch.Generator(device=dev).manual_seed(3)
    qkv = torch.randn(T + 1, 3 * H, D, generator=g, device=dev).half()
    q, k, v = qkv[:T, :H], qkv[:T, H : 2 * H], qkv[:T, 2 * H :]
    pages = torch.randn(2, 3, H, PAGE_TOKENS, D, generator=g, device=dev).half()
    scheme, pos = Vanilla(theta=1e4, head_dim=D), torch.arange(T, device=dev)
    slots, ints = pos.int() + PAGE_TOKENS, (_i32([[1]], dev), _i32([T], dev), _i32([0, T], dev))
    four = lambda x: x.transpose(0, 1)[None]  # noqa: E731
    before, kept = qkv.clone(), pages.clone()
    for out in (qkv[1:, :H], k, qkv[:T, 1 : H + 1], pages[0, 1].transpose(0, 1)[:T]):
        if out.data_ptr() != pages[0, 1].data_ptr():
            with pytest.raises(ValueError, match="overlap"):
                rope_axes(four(q), four(k), pos, scheme, out=(four(out), None))
        with pytest.raises(ValueError, match="overlap"):
            paged_append(k, v, pages[0], pages[1], slots, q=q, positions=pos, scheme=scheme, q_out=out)
        if out.data_ptr() != k.data_ptr():
            with pytest.raises(ValueError, match="overlap"):
                paged_attention(q, pages[0], pages[1], *ints, out=out)
    with pytest.raises(ValueError, match="overlap"):
        rope_axes(four(q), four(k), pos, scheme, out=(four(q), four(q)))
    with pytest.raises(ValueError, match="overlap"):
        paged_append(k, v, pages[0], pages[0], slots)
    assert torch.equal(qkv, before) and torch.equal(pages, kept)
    want = rope_axes(four(q), four(k), pos, scheme)
    rope_axes(four(q), four(k), pos, scheme, out=(four(q), four(k)))
    assert torch.equal(four(q), want[0]) and torch.equal(four(k), want[1]) and torch.equal(v, before[:T, 2 * H :])
    qkv.copy_(before)
    paged_append(k, v, pages[0], pages[1], slots, q=q, positions=pos, scheme=scheme, q_out=q)
    assert torch.equal(four(q), want[0]) and torch.equal(pages[0, 1].transpose(0, 1)[:T], want[1][0].transpose(0, 1))
    # tokens of one page to another
    paged_append(pages[0, 1].transpose(0, 1), pages[1, 1].transpose(0, 1), pages[0], pages[1], torch.arange(128, 192, device=dev).int())
    assert torch.equal(pages[:, 2], pages[:, 1])
    paged_attention(q, pages[0], pages[1], *ints, out=k)


def test_slots_outputs_over_other_memory_are_refused(dev):
    m = torch.zeros(64, dtype=torch.int32, device=dev)
    lens, new, table, free, ring = m[:2], m[2:4], m[4:10].view(2, 3), m[10:14], m[14:16]
    free.copy_(_i32([1, 2, 3, 4], dev))
    ring[1], new[0] = 4, 3
    fresh = m[20:]
    names = ("table", "lens", "starts", "slots", "positions", "ring", "status")
    for name, over in (("slots", lens), ("positions", new), ("status", ring[:1]), ("lens", free[:2]), ("starts", fresh[7:10]), ("table", m[5:11])):
        parts = dict(zip(names, fresh.split([6, 2, 3, 2, 2, 2, 1, 26])))
        parts[name] = over.view(2, 3) if name == "table" else over
        with pytest.raises(ValueError, match="overlap"):
            page_slots(lens, new, table, free, ring, 2, out=PageSlots(**parts))
    parts = dict(zip(names, fresh.split([6, 2, 3, 4, 4, 2, 1, 22])), table=table)
    got = page_slots(lens, new, table, free, ring, 4, out=PageSlots(**parts)).check()
    assert got.slots.tolist() == [64, 65, 66, -1] and table.tolist() == [[1, 0, 0], [0, 0, 0]] and got.ring.tolist() == [1, 3]


def test_rotation_of_more_workgroups_than_a_launch_has(dev):
    """Rows that are not 16-byte aligned, four to a workgroup, past 2^32 threads: every row is turned, once."""
    D, S = 128, 2**26 + 9
    scheme = Vanilla(theta=1e4, head_dim=D)
    buf = torch.ones(S * D + 1, dtype=BF16, device=dev)
    x = buf[1:].view(1, 1, S, D)
    pos = torch.full((1,), 3, device=dev).expand(S)
    one = rope_axes(torch.ones(1, 1, 1, D, dtype=BF16, device=dev), None, pos[:1], scheme)[0]
    rope_axes(x, None, pos, scheme, out=(x, None))
    for at in range(0, S, 2**22):
        assert bool((x[:, :, at : at + 2**22] == one).all()), at
    assert buf[0] == 1


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Hq,Hkv,n,L,others", [(70, 8, 2, 200, 3000, 1), (64, 2, 2, 900, 2000, 1), (64, 8, 2, 193, 193, 1), (70, 8, 2, 70, 3000, 0), (300, 4, 1, 300, 1500, 0), (257, 2, 2, 257, 2000, 0)])
def test_attention_of_a_chunk_among_decoding_rows(dev, B, Hq, Hkv, n, L, others, dtype):
    """Many rows of one token, or of none, and one of many: few matrix rows a row on average."""
    D = 64
    g = torch.Generator(device=dev).manual_seed(B)
    lens, new = [(53 * i) % 200 + 1 for i in range(B)], [others] * B
    lens[B // 2], new[B // 2] = L, n
    k, v, table = _pages(g, dev, lens, Hkv, D, dtype, junk=math.nan)
    starts = _starts(new)
    q = torch.randn(starts[-1], Hq, D, generator=g, device=dev).to(dtype)
    for mask in ("bottom_right", "none"):
        want, tol = _reference(q, k, v, table, lens, starts, 1 / math.sqrt(D), mask)
        got = paged_attention(q, k, v, table, _i32(lens, dev), _i32(starts, dev), mask=mask)
        _check(got, want, tol, mask)


@pytest.mark.parametrize("scheme", [Vanilla(theta=1e6, head_dim=128), Llama3(theta=5e5, head_dim=128, factor=8.0),
                                    Proportional(theta=1e6, head_dim=128, partial_rotary_factor=0.25), MRope(theta=1e6, head_dim=128)])
def test_eviction_turns_keys_that_rope_axes_rotated(dev, scheme):
    """One axis, all channels paired i and i + D / 2: the cache's tables turn such keys to their new positions."""
    H, S, D = 2, 300, 128
    g = torch.Generator(device=dev).manual_seed(6)
    k = torch.randn(1, H, S, D, generator=g, device=dev)
    old = torch.arange(S, device=dev)
    keep = torch.randperm(S, generator=g, device=dev)[:100].sort().values
    rotated = rope_axes(None, k, old, scheme)[1]
    tables = [*scheme.host_cos_sin(old.cpu(), F32), *scheme.host_cos_sin(torch.arange(100), F32)]
    got, _ = rerope_gather(rotated, None, keep, *tables)
    want = rope_axes(None, k[:, :, keep].contiguous(), torch.arange(100, device=dev), scheme)[1]
    # the tables' angles are fp32 products of at most 300 (2^-24 of it each, the inverse frequency's as well: 2^-15 over three
    # rotations), turning a pair by as much of its length, at most 12 of N(0, 1)'s pairs here
    assert float((got - want).abs().max()) <= 2.0**-15 * 12


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,new", [([70, 200], [1, 1]), ([400, 130], [100, 90]), ([3000], [300])])
def test_queries_whose_scores_are_all_minus_infinity(dev, lens, new, dtype):
    """They get zeros, as those that see no key, and a row beside them what it gets alone."""
    H, D = 2, 128
    g = torch.Generator(device=dev).manual_seed(8)
    k, v, table = _pages(g, dev, lens, H, D, dtype)
    starts = _starts(new)
    q = torch.randn(starts[-1], H, D, generator=g, device=dev).to(dtype)
    q[..., 5] = 1.0
    k[:, 0, :, 5] = 0.0
    want = paged_attention(q, k, v, table, _i32(lens, dev), _i32(starts, dev))
    k[:, 1, :, 5] = -math.inf
    got = paged_attention(q, k, v, table, _i32(lens, dev), _i32(starts, dev))
    assert not got[:, 1].any() and torch.equal(got[:, 0], want[:, 0])
