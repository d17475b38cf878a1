"""Sizes and refusals of the typed operators at the edges of what they accept, without a GPU."""
import pytest

pytest.importorskip("torch")
import test_cpu_typed_ops as base  # noqa: E402


@pytest.fixture(scope="module")
def L(eg2):
    return eg2._lib


@pytest.mark.parametrize("n", [1, 9, 4097, 100003, 1 << 24, 1 << 30])
@pytest.mark.parametrize("d", [1, 512, 4099, 700000, 1 << 20])
def test_embed_rows_grad_workspace_of_many_wide_rows(L, n, d):
    """16 bytes an item and two rows a chunk; the chunks are at most a share for each of
    1184 warps of 256 columns, and one more."""
    size = L.load().eg2_embed_rows_grad_workspace(n, d)
    fixed = (1 << 20) + 128 * 1024 * 4 + 8 * 256  # flags, histogram, padding
    assert 16 * n < size <= 16 * n + 8 * d * (1184 // -(-d // 256) + 1) + fixed
