"""Products and gradients of few tiles on either side of the numbers up to which a tile's sum is split over clusters of eight,
four and two, and about the depths at which pairs of CTAs hand over to single ones."""
import pytest
import torch

from mx_reference import E2M1, E4M3, decode, random_codes
from test_gpu_mx import check_grad, check_product, close, ops

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


@pytest.mark.parametrize("across", [False, True])
@pytest.mark.parametrize("m,n,k", [(128, 1024, 1280), (128, 1024, 1728), (128, 1024, 1792), (256, 2048, 1472), (256, 2048, 1600),
                                   (128, 1056, 960), (128, 1056, 1024), (1000, 992, 1728), (1000, 992, 1800)])
def test_gradients_about_the_depths_where_single_blocks_take_over(m, n, k, across):
    """24 steps saved by splitting where a row's scales lie on four bytes, 14 where they do not"""
    check_grad(m, n, k, E4M3, across, seed=k)


def test_gradients_with_scales_off_four_bytes():
    """the choice goes by where scale bytes lie, too; both kernels hold the same bound"""
    m, n, k = 256, 512, 1280
    c, s = random_codes(k, n, E4M3, 1)
    g = torch.randn(m, k, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    w = decode(c, s, E4M3)
    exact, size = g.double() @ w, g.double().abs() @ w.abs()
    base = torch.zeros(s.numel() + 1, dtype=torch.uint8, device="cuda")
    base[1:] = s.reshape(-1).cuda()
    for scales in (s.cuda(), base[1:].view(s.shape)):
        close(ops().mx_matmul_grad(g.cuda(), c.cuda(), scales, m, n, k, E4M3, False), exact, size, k, 16)
