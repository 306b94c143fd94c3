"""Edges of the operators over a table: small rows, far-apart and tiny values, mixed memory, streams, the largest tiles and several pieces.
References in 64 bits; the bounds are those of test_gpu_table.py, whose docstring derives them."""
import pytest

import arrowspace_amd as A

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_table import _check4, _plain4  # noqa: E402


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40])
def test_scores4_of_short_aligned_f16_rows(d, zeros):
    """Rows of less than a step of 32 columns, read from memory as they lie."""
    for m in (5, 9, 16):
        for v in (1, 17, 300):
            codes, s, z, w = _plain4(v, d, 32, "f16", zeros, m + v + d)
            t = A.Table4.from_codes(codes, s, z, dim=d, group=32)
            x = torch.randn(m, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(m)).half()
            _check4(t, w, x)
            wide = torch.full((m, d + 8), float("nan"), device="cuda", dtype=torch.float16)
            wide[:, :d] = x
            assert torch.equal(t.scores(wide[:, :d]), t.scores(x))
