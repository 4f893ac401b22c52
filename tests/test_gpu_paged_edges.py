"""The paged attention where its numbers are hard, against softmaxes in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from fade_amd.kernels import paged_attention
from fade_amd.pages import PAGE_TOKENS
from test_gpu_paged import BF16, F16, _check, _i32, _pages, _starts

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
