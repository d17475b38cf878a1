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


@pytest.mark.parametrize("heads", [(8, 0, 0), (4, 2, 2), (32, 0, 0), (1, 0, 65536)])
def test_qkv_norm_rope_refuses_rows_past_2_to_33(L, heads):
    """Rows of all heads together: the grid's counts are sized for fewer than 2^33, both ways."""
    kw = dict(n=1 << 30, q_heads=heads[0], k_heads=heads[1], v_heads=heads[2], d=2)
    apart, same = L.Strides3(*[(1 << 20, 2)] * 3), L.Strides3(*[(0, 0)] * 3)
    assert base.qkv(L, **kw, out_stride=apart, x_stride=same) == base.INVALID
    assert base.qkv_grad(L, **kw, dx_stride=apart, dout_stride=same, x_stride=same) == base.INVALID
