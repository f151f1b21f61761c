"""Products and gradients of few tiles on either side of the numbers up to which a tile's sum is split over clusters of eight,
four and two."""
import pytest
import torch

from mx_reference import E2M1, E4M3
from test_gpu_mx import check_grad, check_product

pytestmark = pytest.mark.gpu
TILES = [15, 16, 18, 32, 34, 37, 74, 75]


@pytest.mark.parametrize("fmt", [E4M3, E2M1])
@pytest.mark.parametrize("tiles", TILES)
@pytest.mark.parametrize("m,k", [(1, 4096), (128, 4096)])
def test_products(m, k, tiles, fmt):
    check_product(m, 128 * tiles - 3, k, fmt, fmt, seed=tiles, bias=True)


@pytest.mark.parametrize("tiles", TILES)
@pytest.mark.parametrize("m,k,across", [(128, 4096, False), (127, 2048, True)])
def test_gradients(m, k, across, tiles):
    first = check_grad(m, 128 * tiles - 32 * (tiles % 2), k, E4M3, across, seed=tiles)
    assert torch.equal(first, check_grad(m, 128 * tiles - 32 * (tiles % 2), k, E4M3, across, seed=tiles))
