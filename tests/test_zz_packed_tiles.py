"""Packed products of more rows than a workgroup streams."""
import pytest
import torch

from .test_gpu_packed import BF16, DEV, F32, INT8, close, definition, gen, pack, rounded, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [INT8, BF16])
@pytest.mark.parametrize("M", [1, 40, 700])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_and_results_in_columns_of_one_buffer(M, dtype, kind):
    from burn_dragon_amd.packed import grouped_product, product

    K, N, g = 128, 200, gen(M)
    x, w = rows_of(g, M, K, dtype), torch.randn((K, N), generator=g)
    packed = pack(w, kind)
    want, bound = definition(x, w, kind)
    for at, to in ((0, K), (N + 5, 3)):
        wide = torch.full((M, K + N + 8), 7.0, device=DEV, dtype=dtype)
        wide[:, at:at + K] = x.to(DEV, dtype)
        before = wide.clone()
        out = product(wide[:, at:at + K], packed, out=wide[:, to:to + N])
        close(out, want, rounded(bound, want, dtype))
        close(grouped_product(wide[:, at:at + K], packed, [0, M], out=wide[:, to:to + N]), want, rounded(bound, want, dtype))
        wide[:, to:to + N] = 7.0
        assert torch.equal(wide, before)
        with pytest.raises(Exception, match="overlaps"):
            product(wide[:, at:at + K], packed, out=wide[:, 8:8 + N])
