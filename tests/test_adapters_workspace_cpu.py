"""The workspace of the adapters' gradients holds what the call writes there and no more."""
import pytest

from jmodt_amd import _lib as L


def up(n):
    return (n + 255) // 256 * 256


@pytest.mark.parametrize("m,k,n,rank,adapters", [(0, 8, 4, 2, 3), (1, 512, 512, 16, 1), (512, 1024, 1024, 64, 64), (513, 512, 256, 16, 4), (4096, 512, 512, 16, 8), (16383, 96, 80, 64, 3),
                                                 (16384, 96, 80, 64, 3), (131072, 512, 512, 64, 4), (1 << 20, 256, 256, 128, 1023)])
@pytest.mark.parametrize("kind,size", [(0, 4), (1, 2), (2, 2)])
def test_size(m, k, n, rank, adapters, kind, size):
    """u (m, rank) float32 always, one row at least; partials per chunk of rows beyond 512 rows (512, above 8192 rows; else 128 or 256); both
    weights transposed from 16384 rows on"""
    want = up(4 * max(m, 1) * rank)
    if m >= 16384:
        want += up(adapters * rank * k * size) + up(adapters * rank * n * size)
    if m > 512:
        chunk = 512 if m > 8192 else 128 if m <= 4096 else 256
        want += (-(-m // chunk) + min(adapters, m)) * rank * (k + n) * 4
    assert L.load().jm_adapter_grad_workspace_bytes(m, k, n, rank, adapters, kind) == want
