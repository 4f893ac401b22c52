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
