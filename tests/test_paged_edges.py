"""What the paged operators' entry points refuse, on the CPU."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from fade_amd import _lib


def test_forward_mode_is_refused():
    x = torch.ones(3, dtype=torch.float16)
    with forward_ad.dual_level():
        _lib.no_gradient("op", x, None)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for context in (torch.enable_grad(), torch.no_grad()):
            with context, pytest.raises(ValueError, match="op: has no forward-mode derivative"):
                _lib.no_gradient("op", None, x, dual)
        _lib.no_gradient("op", forward_ad.unpack_dual(dual).primal)
    _lib.no_gradient("op", x)


def test_places_of_an_output():
    x = torch.zeros(4, 3, 8)
    rows = torch.zeros(64)
    for t in (x, x.transpose(0, 1), x[::2, :, 1:5], x[:0], x[:1].expand(1, 3, 8), rows.as_strided((2, 3, 8), (24, 8, 1)),
              rows.as_strided((1, 3, 8), (0, 8, 1)), rows.as_strided((2, 1, 8), (9, 3, 1)), x[:0].expand(0, 3, 8)):
        assert _lib.each_once(t), t.stride()
    for t in (x[:1].expand(4, 3, 8), x[:, :1].expand(4, 3, 8), rows.as_strided((3, 3, 8), (4, 12, 1)), rows.as_strided((2, 3, 8), (16, 8, 1))):
        assert not _lib.each_once(t), t.stride()
