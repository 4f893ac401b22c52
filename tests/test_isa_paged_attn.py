"""The paged attention's LDS DMAs respect the issue hazards that the hardware does not interlock and
that the compiler cannot see inside inline asm (CPU only: hipcc cross-compiles)."""

import os
import subprocess

import pytest

from test_isa_lds_dma_hazards import CSRC, FLAGS, HIPCC, hazards

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")


def test_lds_dma_hazard_free(tmp_path):
    out = tmp_path / "paged_attn.s"
    subprocess.run([HIPCC, *FLAGS, os.path.join(CSRC, "paged_attn.hip"), "-o", str(out)], check=True, capture_output=True, timeout=900)
    n, bad = hazards(out.read_text())
    assert n > 0, "no LDS DMA found"
    assert not bad, f"{len(bad)} of {n} LDS DMAs break an issue hazard, e.g. {bad[:3]}"
