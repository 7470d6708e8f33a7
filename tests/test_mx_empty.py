"""Quantised caches that hold nothing (no rows, no pages, no positions) on the CPU: a server before its first request."""
import pytest
import torch

from palu_tt.cache import LatentCache, MXCache


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("role", ["k", "v"])
@pytest.mark.parametrize("shape", [(0, 2, 64, 64), (3, 0, 32, 96), (2, 1, 0, 32)], ids=str)
def test_empty_caches(fmt, role, shape):
    rows = torch.zeros(shape, dtype=torch.bfloat16)
    assert tuple(LatentCache.from_rows(rows, role).to_rows().shape) == shape
    for c in (MXCache.zeros(*shape, "cpu", role, fmt), MXCache.from_rows(rows, role, fmt)):
        codes, scales = c.parts()
        assert c.shape == shape == tuple(c.to_rows().shape) == tuple(codes.shape) and c.to_rows().dtype == torch.bfloat16
        assert tuple(scales.shape) == (*shape[:3], shape[3] // 32) and c.nbytes() == 0
