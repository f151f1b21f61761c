"""The layer on microscaled operands where values are not ordinary ones, against the quantisers' definition in 64 bits: the
scale of a group is the largest power of two that keeps its largest magnitude within the format's largest value, its
byte limited to 0 ... 254 before the codes are made; a group of zeros has byte 127, one that holds an infinity or a NaN stands
for NaN as a whole.  Tolerances are those of the products: one rounding to bfloat16 after sums in binary32."""
import numpy as np
import pytest
import torch

import mx_reference as R
from test_gpu_mx import STEP, close, values

pytestmark = pytest.mark.gpu
FORMATS = {"e4m3": R.E4M3, "e5m2": R.E5M2, "e2m1": R.E2M1}
LARGEST = {R.E4M3: (8, 1.75), R.E5M2: (15, 1.75), R.E2M3: (2, 1.875), R.E2M1: (2, 1.5)}   # c * 2^top
GRID = {R.E4M3: (3, -6), R.E5M2: (2, -14), R.E2M3: (3, 0), R.E2M1: (1, 0)}                # mantissa bits, smallest exponent


def quantised(x, fmt, group=32):
    """(values, scale bytes) in float64 and uint8 that a [rows, cols] tensor is quantised to"""
    g = x.detach().double().cpu().numpy().reshape(x.shape[0], -1, group)
    top, c = LARGEST[fmt]
    mant, lowest = GRID[fmt]
    finite = np.isfinite(g).all(2)
    g = np.where(finite[:, :, None], g, 0.0)
    amax = np.abs(g).max(2)
    m, e = np.frexp(amax)                                     # amax = m * 2^e, m in [1/2, 1)
    s = np.where(amax > 0, np.clip(e - 1 - top + (2 * m > c) + 127, 0, 254), 127)
    q = np.ldexp(g, (127 - s)[:, :, None])
    step = np.maximum(np.frexp(np.abs(q))[1] - 1, lowest) - mant
    v = np.ldexp(np.round(np.ldexp(q, -step)), step + (s - 127)[:, :, None])          # ties to even
    v = np.where(finite[:, :, None], v, np.nan)
    return torch.from_numpy(v.reshape(x.shape)), torch.from_numpy(np.where(finite, s, 255).astype(np.uint8))


def product(a, b):
    """a @ b.T and the sum of magnitudes, NaN wherever a row of either holds one"""
    a0, b0 = a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0)
    bad = torch.isnan(a).any(1)[:, None] | torch.isnan(b).any(1)[None]
    return torch.where(bad, float("nan"), a0 @ b0.t()), a0.abs() @ b0.abs().t()


def check_step(x, w, b, g, name):
    """y, dx, dw of a step, and the serving form's y"""
    from mor_b200.nn import MXLinear, mx_linear
    f = FORMATS[name]
    (m, k), n = x.shape, w.shape[0]
    xd, wd, bd, gd = (t.to(torch.bfloat16).cuda() for t in (x, w, b, g))
    xd.requires_grad_(), wd.requires_grad_()
    y = mx_linear(xd, wd, bd, f)
    dx, dw = torch.autograd.grad(y, (xd, wd), gd)
    xq, wq = quantised(xd, f)[0], quantised(wd, f)[0]
    g64, b64 = gd.double().cpu(), bd.double().cpu()
    exact, size = product(xq, wq)
    close(y.detach(), exact + b64, size + b64.abs(), k, STEP[f])
    # The gradients take the quantised values as bf16, exact but below 2^-126, where each is off by half a step of 2^-133 at
    # most: that times what it meets is added to the size that `close` multiplies by (n / 16 + 9) 2^-23 > 2^-20.
    for got, (a, q), terms in ((dx, (g64, wq.t()), n), (dw, (g64.t(), xq.t()), m)):
        exact, size = product(a, q)
        close(got, exact, size + a.abs().sum(1, keepdim=True) * 2.0 ** (-134 + 20), terms, 16)
    layer = MXLinear(k, n, device="cuda", elem_format=name)
    with torch.no_grad():
        layer.weight.copy_(wd), layer.bias.copy_(bd)
    served = layer.pack()(xd)
    assert torch.equal(torch.isnan(served), torch.isnan(y)) and torch.equal(served.nan_to_num(nan=0.0), y.detach().nan_to_num(nan=0.0))


def operands(m, n, k, seed):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=gen), 0.02 * torch.randn(n, k, generator=gen), torch.randn(n, generator=gen),
            torch.randn(m, n, generator=gen), gen)


SIZES = [(1, 8, 32), (9, 40, 96), (70, 72, 512), (300, 264, 1024)]


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_value_that_is_no_number_spoils_its_group(value, m, n, k, name):
    """one in an input: its row of y and its group's columns of the weight's gradient are NaN, the rest is as without it"""
    x, w, b, g, gen = operands(m, n, k, m)
    x[m // 2, int(torch.randint(0, k, (1,), generator=gen))] = value
    check_step(x, w, b, g, name)


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_values_that_are_no_numbers_among_ordinary_ones(m, n, k, name):
    """several in either operand, a group of nothing else, and one among zeros"""
    _, w, b, g, gen = operands(m, n, k, m + 1)
    x = values("bad", m, k, m, torch.float32)
    if m > 5:
        x[4, :32] = float("nan")
        x[5, 32:64] = 0.0
        x[5, 40] = float("inf")
    w[n // 2, k - 1], w[n - 1, 0] = float("-inf"), float("nan")
    check_step(x, w, b, g, name)


@pytest.mark.parametrize("fmt", [R.E4M3, R.E5M2, R.E2M3])
@pytest.mark.parametrize("group", [8, 32, 256])
def test_operand_groups_that_hold_no_numbers(fmt, group):
    """byte 255 and codes of zero for these groups, the others exactly as they are without"""
    import mor
    x = values("normal", 37, 768, 7, torch.bfloat16)
    want = mor.ops.quantize_mx(x.cuda(), 37, 768, group, fmt)
    spoiled = values("bad", 37, 768, 7, torch.bfloat16)
    spoiled[3] = float("nan")
    got = mor.ops.quantize_mx(spoiled.cuda(), 37, 768, group, fmt, operand=True)
    bad = (~torch.isfinite(spoiled)).reshape(37, -1, group).any(2)
    assert torch.equal(got[1].cpu(), torch.where(bad, 255, want[1].cpu()))
    assert torch.equal(got[0].cpu(), torch.where(bad.repeat_interleave(group, 1), 0, want[0].cpu()))


# ------------------------------------------------------------------------------------------------ very small and large groups
@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("power", [-80, -100, -110, -114, -116, -120, -122, -126, -130])
def test_small_groups(power, m, n, k, name):
    """down to where the scale's byte is 0 and to subnormal inputs, zeros among them; the other operand large, so that the
    products are ordinary numbers"""
    x, w, b, g, gen = operands(m, n, k, m)
    zeros = torch.rand(m, k, generator=gen) < 0.2
    x[zeros] = 0.0
    up, down = 2.0 ** 60, 2.0 ** power
    check_step(x * down, w * up, b * down * up, g * up, name)
    check_step(w * down, x * up, g[:, 0] * down * up, g.t() * up, name)


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("kind,w_scale", [("tiny", 2.0 ** 60), ("huge", 2.0 ** -60), ("ties", 1.0), ("sparse", 1.0)])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_values_of_every_size(m, n, k, kind, w_scale, name):
    _, w, b, g, _ = operands(m, n, k, m)
    check_step(values(kind, m, k, m, torch.float32), w * w_scale, b, g * w_scale, name)


@pytest.mark.parametrize("fmt", [R.E4M3, R.E5M2, R.E2M3])
@pytest.mark.parametrize("group", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("kind", ["normal", "wide", "tiny", "huge", "ties", "sparse", "bad"])
def test_operands_are_the_nearest_values(kind, group, fmt):
    """scale bytes and values by the definition, bit for bit; the number of vectors is no multiple of a warp's"""
    import mor
    x = values(kind, 37, 768, 11, torch.bfloat16)
    if kind == "tiny":
        x[20:] *= 2.0 ** torch.linspace(0, 60, 17)[:, None]
        x[:, ::5] = 0.0
    codes, scales = mor.ops.quantize_mx(x.cuda(), 37, 768, group, fmt, operand=True)
    want, bytes_ = quantised(x, fmt, group)
    assert torch.equal(scales.cpu(), bytes_)
    got = R.decode(codes, scales, fmt, group)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])
    assert not bool(codes.cpu()[nan].any())


@pytest.mark.parametrize("fmt", [R.E4M3, R.E5M2, R.E2M3])
def test_operands_of_ordinary_groups_keep_their_bytes(fmt):
    """with and without the mode alike, at sizes of one group up to more than a round of blocks, and nothing behind them"""
    import mor
    from mor_b200 import cabi
    for rows, cols in ((1, 32), (3, 32), (129, 96), (1000, 4128)):
        x = (torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows)) * 3).to(torch.bfloat16).cuda()
        want = mor.ops.quantize_mx(x, rows, cols, 32, fmt)
        got = [torch.full((t.numel() + 512,), 9, dtype=torch.uint8, device="cuda") for t in want]
        cabi.call("mor_b200_quantize_mx", x.data_ptr(), got[0].data_ptr(), got[1].data_ptr(), rows, cols, 32, fmt + cabi.MX_OPERAND,
                  torch.cuda.current_stream().cuda_stream)
        for u, v in zip(got, want):
            assert torch.equal(u[:v.numel()].view(v.shape), v) and bool((u[v.numel():] == 9).all())
