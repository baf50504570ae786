"""CPU tensors in 16 bits through the token-model operators: sums in fp32, rounded once, as on a GPU.

Tolerance: half a step of the type for the one rounding, and 2^-24 of the sum of magnitudes for each of up to 2000 fp32 additions,
which is 2000 * 2^-24 = 1.2e-4 of it."""
import pytest
import torch

from distributed_tensorflow_amd.ops import embedding


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_frequent_id(dtype):
    g = torch.Generator().manual_seed(1)
    table = torch.randn(5, 3, generator=g).to(dtype)
    ids = torch.where(torch.rand(2000, generator=g) < 0.9, 2, 4)
    ids[::50], ids[1::50] = -1, 5
    up = torch.rand(2000, 3, generator=g).to(dtype)
    sums, sizes = torch.zeros(5, 3, dtype=torch.float64), torch.zeros(5, 3, dtype=torch.float64)
    keep = (ids >= 0) & (ids < 5)
    sums.index_add_(0, ids[keep], up[keep].double())
    sizes.index_add_(0, ids[keep], up[keep].double().abs())

    def near(got, want, size):
        assert got.dtype == dtype
        assert bool(((got.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 1.2e-4 * size).all())

    leaf = table.clone().requires_grad_(True)
    out = embedding.embedding_lookup(leaf, ids, 0.5)
    near(out.detach(), 0.5 * table.double()[ids.clamp(0, 4)] * keep[:, None], torch.zeros(1))
    near(torch.autograd.grad(out, leaf, up)[0], 0.5 * sums, 0.5 * sizes)
    after = embedding.update_rows(table.clone(), ids, up, torch.tensor([0.25]), 0.5)
    near(after, table.double() - 0.125 * sums, 0.125 * sizes + table.double().abs())
    for row in (0, 1, 3):
        assert torch.equal(after[row], table[row])
