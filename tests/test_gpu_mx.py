"""Operators on microscaled operands against their definition in 64 bits.

Quantisation and reading back are exact, so bytes and values have to be equal.  A product rounds to bfloat16 once (half a
step, 2^-8 of the value) after sums in binary32: each instruction of the tensor core adds 16 (bf16), 32 (8-bit) or 64
(4-bit) products to the accumulator and may drop what lies below 2^-23 of the running magnitude, which is at most S =
sum |a_k b_k|; eight more such steps stand for the alignment of the products among themselves, the sum over a cluster and
the bias.  So |got - exact| <= 2^-8 |exact| + (K / step + 8 + 1) 2^-23 S (1 + 2^-8).
"""
import math

import numpy as np
import pytest
import torch

import mx_reference as R
from mx_reference import E2M1, E2M3, E4M3, E5M2

pytestmark = pytest.mark.gpu
STEP = {E4M3: 32, E5M2: 32, E2M1: 64}


def ops():
    import mor
    return mor.ops


def close(got, exact, s, k, step):
    got = got.double().cpu()
    assert got.shape == exact.shape
    nan = torch.isnan(exact)
    assert torch.equal(torch.isnan(got), nan)
    tol = 2.0 ** -8 * exact.abs() + (math.ceil(k / step) + 9) * 2.0 ** -23 * s * (1 + 2.0 ** -8) + 2.0 ** -133
    off = torch.where(nan, 0.0, (got - exact).abs() - tol)
    assert bool((off <= 0).all()), f"{int((off > 0).sum())} of {off.numel()} outside, worst {float(off.max()):.3g} at {np.unravel_index(int(off.argmax()), off.shape)}"


# ------------------------------------------------------------------------------------------------ quantisation
def values(kind, rows, cols, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if kind == "wide":
        x = x * 10.0 ** (torch.rand(rows, cols, generator=g) * 60 - 30)
    if kind == "tiny":      # subnormals of either type, and groups below the smallest scale
        x = x * 2.0 ** -130
    if kind == "huge":
        x = x.clamp(-3.9, 3.9) * 2.0 ** 125
    if kind == "ties":      # halfway between codes, under scales of every kind
        x = torch.randint(-24, 25, (rows, cols), generator=g) * 0.25 * 2.0 ** torch.randint(-20, 20, (rows, 1), generator=g)
    if kind == "sparse":
        x = torch.where(torch.rand(rows, cols, generator=g) < 0.97, torch.zeros(()), x)
        x[0, :32] = -0.0
    if kind == "bad":
        x.view(-1)[torch.randint(0, x.numel(), (5,), generator=g)] = float("nan")
        x.view(-1)[torch.randint(0, x.numel(), (5,), generator=g)] = float("inf")
        x.view(-1)[torch.randint(0, x.numel(), (5,), generator=g)] = float("-inf")
    return x.to(dtype)


def check_fp4(x_dev, what=""):
    payload, scales = ops().quantize_mx_fp4(x_dev, x_dev.shape[0], x_dev.shape[1], 32)
    ep, es = R.quantize_fp4(x_dev.double().cpu().numpy())
    assert payload.dtype == torch.uint8 and scales.dtype == torch.uint8
    assert torch.equal(scales.cpu(), es), what
    assert torch.equal(payload.cpu(), ep), what


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["normal", "wide", "tiny", "huge", "ties", "sparse", "bad"])
def test_quantize_fp4_values(kind, dtype):
    check_fp4(values(kind, 37, 224, 1, dtype).cuda(), kind)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (2, 64), (3, 96), (255, 4128), (1024, 2048), (5000, 32)])
def test_quantize_fp4_shapes(rows, cols, dtype):
    check_fp4(values("normal", rows, cols, rows + cols, dtype).cuda())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_fp4_strides(dtype):
    wide = values("normal", 70, 512, 3, dtype).cuda()
    check_fp4(wide[:, 64:288], "slice of columns")
    check_fp4(wide[:, 1:65], "slice off the 16-byte grid")
    check_fp4(wide[::3, 32:96], "every third row")
    check_fp4(wide.t()[:, :64], "transposed")
    check_fp4(wide[:, ::2], "every second column")
    check_fp4(wide[:1].expand(9, 512), "one row repeated")
    check_fp4(values("normal", 64, 65, 4, dtype).cuda()[:, :64], "odd pitch")


@pytest.mark.parametrize("fmt,group", [(E4M3, 32), (E4M3, 8), (E5M2, 32), (E5M2, 256), (E2M3, 32), (E2M1, 32), (E2M1, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dequantize_every_code_under_every_scale(fmt, group, dtype):
    width = R.FORMATS[fmt][0]
    codes = np.tile(np.arange(256, dtype=np.uint8) & ((1 << width) - 1), (256, 1))
    scales = torch.arange(256, dtype=torch.uint8)[:, None].expand(256, 256 // group).contiguous()
    payload = torch.from_numpy(R.pack4(codes) if fmt == E2M1 else codes)
    got = ops().dequantize_mx(payload.cuda(), scales.cuda(), 256, 256, group, fmt, dtype).cpu()
    exact = R.decode(payload, scales, fmt, group)
    want = exact.to(torch.float32).to(dtype)      # one rounding: the values are exact in binary32 or overflow it
    assert got.dtype == dtype
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(nan=1.0, posinf=2.0, neginf=-2.0), want.nan_to_num(nan=1.0, posinf=2.0, neginf=-2.0))


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 64), (3, 96), (777, 2080), (0, 64)])
@pytest.mark.parametrize("fmt", [E4M3, E5M2, E2M1])
def test_dequantize_shapes(rows, cols, fmt):
    p, s = R.random_codes(rows, cols, fmt, 5)
    got = ops().dequantize_mx(p.cuda(), s.cuda(), rows, cols, 32, fmt)
    assert got.shape == (rows, cols) and got.dtype == torch.bfloat16
    assert torch.equal(got.double().cpu(), R.decode(p, s, fmt))


def test_round_trip_of_the_existing_quantiser():
    """dequantize_mx undoes quantize_mx: the fake-quantised values, where no code is zero under a scale below one"""
    x = values("normal", 64, 512, 9, torch.bfloat16).cuda()
    for fmt in (E4M3, E5M2, E2M3):
        c, s = ops().quantize_mx(x, 64, 512, 32, fmt)
        assert torch.equal(ops().dequantize_mx(c, s, 64, 512, 32, fmt).double().cpu(), R.decode(c, s, fmt))


# ------------------------------------------------------------------------------------------------ products
def product_case(m, n, k, fa, fb, seed, bias):
    a, b = R.random_codes(m, k, fa, seed), R.random_codes(n, k, fb, seed + 1)
    bi = torch.randn(n, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16) if bias else None
    return a, b, bi


def check_product(m, n, k, fa, fb, seed=1, bias=False, a=None, b=None):
    ra, rb, bi = product_case(m, n, k, fa, fb, seed, bias)
    a, b = a or ra, b or rb
    got = ops().mx_matmul(a[0].cuda(), a[1].cuda(), b[0].cuda(), b[1].cuda(), m, n, k, fa, fb, None if bi is None else bi.cuda())
    assert got.dtype == torch.bfloat16
    va, vb = R.decode(*a, fa).cuda(), R.decode(*b, fb).cuda()
    exact, s = va @ vb.t(), va.abs() @ vb.abs().t()
    if bi is not None:
        exact, s = exact + bi.double().cuda(), s + bi.double().abs().cuda()
    close(got, exact.cpu(), s.cpu(), k, STEP[fa])
    return got


@pytest.mark.parametrize("fa,fb", [(E2M1, E2M1), (E4M3, E4M3), (E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)])
@pytest.mark.parametrize("m,n,k", [(128, 128, 256), (128, 128, 32), (256, 384, 1024), (1, 128, 256), (16, 256, 512)])
def test_product_formats(m, n, k, fa, fb):
    check_product(m, n, k, fa, fb)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("m", [1, 2, 7, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200, 255, 257, 300, 513])
def test_product_rows(m, fmt):
    check_product(m, 320, 608, fmt, fmt, seed=m, bias=m % 2 == 1)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("n", [1, 2, 8, 31, 100, 127, 129, 255, 257, 1003])
@pytest.mark.parametrize("m", [3, 40, 130, 700])
def test_product_columns(m, n, fmt):
    check_product(m, n, 416, fmt, fmt, seed=n, bias=True)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("k", [32, 64, 96, 128, 160, 256, 288, 512, 1056, 2048, 2080, 8192])
@pytest.mark.parametrize("m", [1, 20, 260])
def test_product_depths(m, k, fmt):
    check_product(m, 192, k, fmt, fmt, seed=k)


@pytest.mark.parametrize("m,n,k,fmt", [(1, 4096, 4096, E2M1), (24, 4096, 8192, E4M3), (1111, 1003, 2080, E5M2), (2048, 2048, 2048, E2M1),
                                       (2500, 1536, 1024, E4M3), (2305, 1501, 608, E4M3), (2305, 1501, 608, E2M1), (1300, 2056, 32, E2M1),
                                       (1300, 2056, 160, E5M2), (4096, 2048, 4128, E2M1), (1300, 1400, 4096, E4M3), (1300, 1400, 8192, E2M1),
                                       (2300, 2501, 4128, E4M3), (2300, 2504, 8224, E2M1), (1100, 1300, 16384, E5M2), (4096, 300, 512, E2M1), (300, 4096, 512, E4M3)])
def test_product_sizes(m, n, k, fmt):
    check_product(m, n, k, fmt, fmt, bias=True)


@pytest.mark.parametrize("m", [1, 300, 5000])
@pytest.mark.parametrize("fmt", [E2M1, E4M3])
def test_product_every_scale_has_its_place(m, fmt):
    """one group of one row is non-zero at a time, each under a scale of its own: a scale taken from another row or
    group shows as a wrong power of two"""
    n, k = 264, 1024
    p = torch.zeros(n, k // (2 if fmt == E2M1 else 1), dtype=torch.uint8)
    s = torch.randint(110, 140, (n, k // 32), generator=torch.Generator().manual_seed(0), dtype=torch.uint8)
    per = p.shape[1] // (k // 32)
    for r in range(n):
        gi = (r * 7) % (k // 32)
        p[r, gi * per:(gi + 1) * per] = 0x22 if fmt == E2M1 else 0x38   # ones
    check_product(m, n, k, fmt, fmt, b=(p, s))


@pytest.mark.parametrize("m", [3, 300, 10000])
@pytest.mark.parametrize("fmt", [E2M1, E4M3])
def test_product_nan_scales_and_extremes(m, fmt):
    n, k = 200, 512
    a, b, _ = product_case(m, n, k, fmt, fmt, 3, False)
    a[1][1, 2] = 255                 # a NaN group spoils its row of the result and nothing else
    b[1][150, 15] = 255
    a[1][2, :] = 1                   # a row far below the others
    check_product(m, n, k, fmt, fmt, a=a, b=b)
    z = torch.zeros_like(a[0])
    assert not bool(ops().mx_matmul(z.cuda(), torch.full_like(a[1], 127).cuda(), b[0][:100].cuda(), b[1][:100].cuda(), m, 100, k, fmt, fmt).any())


def same_class(got, exact):
    """NaN and infinities where the exact result has them, and nowhere else"""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(exact))
    assert torch.equal(torch.where(torch.isinf(got), got, 0.0), torch.where(torch.isinf(exact), exact, 0.0))


@pytest.mark.parametrize("m", [6, 140, 4000])
@pytest.mark.parametrize("fa,fb", [(E4M3, E4M3), (E5M2, E4M3), (E5M2, E5M2)])
def test_product_codes_that_are_no_number(m, fa, fb):
    n, k = 700, 256
    a, b, _ = product_case(m, n, k, fa, fb, 5, False)
    b[0][:] = torch.where((b[0] & 0x7F) == 0, torch.full_like(b[0], 0x30), b[0])     # no zero meets an infinity
    a[0][1, 3], a[0][m - 1, 200] = 0x7F, 0xFF
    b[0][n - 1, 17] = 0x7F
    if fa == E5M2:
        a[0][3, 100], a[0][4, 101] = 0x7C, 0xFC
    bias = torch.zeros(n, dtype=torch.bfloat16)
    bias[5], bias[6] = float("nan"), float("-inf")
    got = ops().mx_matmul(*(t.cuda() for t in (*a, *b)), m, n, k, fa, fb, bias.cuda())
    same_class(got, (R.decode(*a, fa) @ R.decode(*b, fb).t()) + bias.double())


@pytest.mark.parametrize("across", [False, True])
@pytest.mark.parametrize("m,n,k", [(40, 64, 100), (2400, 1312, 90)])
def test_gradients_that_are_no_number(m, n, k, across):
    """spoil their own rows of the result and nothing else, zeros behind the last k included"""
    g = torch.randn(m, k, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    g[3, 7], g[m - 1, k - 1], g[5, 0], g[6, k - 1] = float("nan"), float("inf"), float("-inf"), float("inf")
    w = R.random_codes(k, n, E4M3, 2)
    w[0][:] = torch.where((w[0] & 0x7F) == 0, torch.full_like(w[0], 0x30), w[0])
    got = ops().mx_matmul_grad((g.t().contiguous() if across else g).cuda(), w[0].cuda(), w[1].cuda(), m, n, k, E4M3, across)
    same_class(got, g.double() @ R.decode(*w, E4M3))


def test_product_empty():
    p, s = R.random_codes(4, 64, E4M3, 0)
    e = torch.empty(0, 64, dtype=torch.uint8), torch.empty(0, 2, dtype=torch.uint8)
    o = ops()
    assert o.mx_matmul(e[0].cuda(), e[1].cuda(), p.cuda(), s.cuda(), 0, 4, 64, 0, 0).shape == (0, 4)
    assert o.mx_matmul(p.cuda(), s.cuda(), e[0].cuda(), e[1].cuda(), 4, 0, 64, 0, 0).shape == (4, 0)
    g = torch.ones(0, 4, dtype=torch.bfloat16).cuda()
    z = o.mx_matmul_grad(g, e[0].cuda(), e[1].cuda(), 4, 64, 0, 0, True)      # no tokens: a gradient of zeros
    assert z.shape == (4, 64) and not bool(z.any())


@pytest.mark.parametrize("m,n,k", [(1, 256, 4096), (40, 512, 4096), (600, 600, 1024), (2400, 2300, 1024), (1300, 1400, 4096)])
def test_product_repeats_bit_for_bit_on_any_stream(m, n, k):
    a, b, _ = product_case(m, n, k, E4M3, E4M3, 8, False)
    args = [t.cuda() for t in (*a, *b)]
    first = ops().mx_matmul(*args, m, n, k, 0, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(6):          # two streams at once
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(ops().mx_matmul(*args, m, n, k, 0, 0))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_first_cuda_call_of_a_thread():
    """a thread that has not touched the device before (autograd's workers) can make the calls"""
    import threading
    a, b, _ = product_case(130, 96, 256, E4M3, E4M3, 4, False)
    args = [t.cuda() for t in (*a, *b)]
    g = torch.randn(130, 96, device="cuda").to(torch.bfloat16)
    calls = (lambda: ops().mx_matmul(*args, 130, 96, 256, 0, 0), lambda: ops().mx_matmul_grad(g, args[2], args[3], 130, 256, 96, 0, False))
    for call in calls:
        want, got = call(), []
        t = threading.Thread(target=lambda: got.append(call()))
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert got and torch.equal(got[0], want)


def test_product_strided_and_offset_operands():
    a, b, _ = product_case(70, 96, 256, E4M3, E4M3, 4, False)
    want = ops().mx_matmul(*(t.cuda() for t in (*a, *b)), 70, 96, 256, 0, 0)
    wide = torch.zeros(70, 300, dtype=torch.uint8, device="cuda")
    wide[:, 7:263] = a[0].cuda()
    base = torch.zeros(96 * 256 + 3, dtype=torch.uint8, device="cuda")
    base[3:] = b[0].cuda().reshape(-1)
    sb = torch.zeros(96 * 8 + 1, dtype=torch.uint8, device="cuda")
    sb[1:] = b[1].cuda().reshape(-1)
    assert torch.equal(ops().mx_matmul(wide[:, 7:263], a[1].cuda(), base[3:].view(96, 256), sb[1:].view(96, 8), 70, 96, 256, 0, 0), want)


def test_rows_beyond_the_result_are_left_alone():
    """the C entry writes [m, n] and nothing after it"""
    from mor_b200 import cabi
    for m, n in ((5, 40), (130, 133), (1, 1), (300, 264), (2305, 1501), (2304, 1032)):
        a, b, _ = product_case(m, n, 96, E4M3, E4M3, 4, False)
        args = [t.cuda() for t in (*a, *b)]
        out = torch.full((m * n + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
        need = cabi.mx_lib().mor_b200_mx_matmul_workspace_bytes(m, n, 96, 0)
        ws = torch.full((need + 64,), 5, dtype=torch.uint8, device="cuda")
        cabi.call("mor_b200_mx_matmul", *(t.data_ptr() for t in args), m, n, 96, 0, 0, None, out.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert bool((out[m * n:] == 7.0).all()) and bool((ws[need:] == 5).all())
        assert torch.equal(out[:m * n].view(m, n), ops().mx_matmul(*args, m, n, 96, 0, 0))


# ------------------------------------------------------------------------------------------------ gradients
def check_grad(m, n, k, fmt, across, seed=1, g=None, w=None):
    gen = torch.Generator().manual_seed(seed)
    if g is None:
        g = torch.randn((k, m) if across else (m, k), generator=gen).to(torch.bfloat16).cuda()
    w = w or R.random_codes(k, n, fmt, seed)
    got = ops().mx_matmul_grad(g, w[0].cuda(), w[1].cuda(), m, n, k, fmt, across)
    assert got.dtype == torch.bfloat16 and got.shape == (m, n)
    gd = (g.t() if across else g).double()
    wd = R.decode(*w, fmt).cuda()
    close(got, (gd @ wd).cpu(), (gd.abs() @ wd.abs()).cpu(), k, 16)
    return got


@pytest.mark.parametrize("across", [False, True])
@pytest.mark.parametrize("fmt", [E4M3, E5M2, E2M3, E2M1])
@pytest.mark.parametrize("m,n,k", [(128, 128, 64), (256, 384, 512), (64, 32, 16)])
def test_grad_formats(m, n, k, fmt, across):
    check_grad(m, n, k, fmt, across)


@pytest.mark.parametrize("across", [False, True])
@pytest.mark.parametrize("fmt", [E4M3, E2M1])
@pytest.mark.parametrize("m", [1, 2, 7, 8, 63, 65, 127, 129, 257, 300])
def test_grad_rows(m, fmt, across):
    check_grad(m, 160, 200, fmt, across, seed=m)


@pytest.mark.parametrize("across", [False, True])
@pytest.mark.parametrize("fmt", [E4M3, E2M1])
@pytest.mark.parametrize("k", [1, 2, 15, 16, 17, 63, 64, 65, 100, 1003, 4096])
def test_grad_depths(k, fmt, across):
    check_grad(136, 288, k, fmt, across, seed=k)


@pytest.mark.parametrize("across", [False, True])
@pytest.mark.parametrize("m,n,k,fmt", [(1000, 2080, 1500, E4M3), (2048, 1024, 4096, E2M1), (4096, 4096, 33, E4M3), (20, 64, 8192, E5M2),
                                       (300, 32, 600, E4M3), (2500, 1056, 640, E2M1), (3000, 2080, 500, E4M3), (2304, 1312, 1000, E2M3),
                                       (2568, 1312, 70, E5M2), (1300, 1408, 2500, E4M3), (2300, 2528, 4001, E2M1), (1304, 1408, 9000, E5M2)])
def test_grad_sizes(m, n, k, fmt, across):
    check_grad(m, n, k, fmt, across)


@pytest.mark.parametrize("fmt", [E4M3, E5M2, E2M3, E2M1])
def test_grad_extreme_scales_and_codes_that_are_no_number(fmt):
    """scales down to 2^-127 make elements that are subnormal in bf16 (rounded there, half a step of 2^-133 at most), scales
    up to 2^100 large ones; columns with an infinity or a NaN in them come out as such and the others do not"""
    k, n, m = 96, 256, 64
    gen = torch.Generator().manual_seed(2)
    c, s = R.random_codes(k, n, fmt, 6)
    s[:, 0::4], s[:, 1::4], s[:, 2::4] = 0, torch.randint(0, 12, (k, 2), generator=gen, dtype=torch.uint8), 227
    if fmt in R.HAS_NAN:
        c[3, 97], c[50, 130] = 0x7F, 0xFF
        if fmt == E5M2:
            c[4, 100], c[5, 140] = 0x7C, 0xFC
    g = (torch.randint(1, 5, (m, k), generator=gen) * torch.where(torch.rand(m, k, generator=gen) < 0.5, -1, 1)).to(torch.bfloat16)
    got = ops().mx_matmul_grad(g.cuda(), c.cuda(), s.cuda(), m, n, k, fmt, False).double().cpu()
    w = R.decode(c, s, fmt)
    exact = g.double() @ w
    t = 2.0 ** -8 * exact.abs() + (math.ceil(k / 16) + 9) * 2.0 ** -23 * (g.abs().double() @ w.abs()) * 1.01 + k * 4 * 2.0 ** -134 + 2.0 ** -133
    fine = torch.isfinite(exact)
    assert torch.equal(torch.isnan(exact), torch.isnan(got)) and torch.equal(exact[~fine & ~torch.isnan(exact)], got[~fine & ~torch.isnan(exact)])
    assert bool(((got - exact).abs()[fine] <= t[fine]).all())


def test_grad_nan_scale_and_strides():
    w = R.random_codes(96, 128, E4M3, 3)
    w[1][5, 2] = 255
    w[0][7, 3] = 0x7F                # a NaN code
    for across in (False, True):
        check_grad(40, 128, 96, E4M3, across, w=w)
    wide = torch.randn(200, 300, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    check_grad(200, 64, 256, E4M3, False, g=wide[:, 40:296])
    check_grad(200, 64, 255, E4M3, False, g=wide[:, 1:256])
    check_grad(77, 64, 200, E4M3, True, g=wide[:, :77])
    check_grad(300, 64, 200, E4M3, False, g=wide.t())
    check_grad(40, 64, 300, E4M3, True, g=wide[:1, :40].expand(300, 40))


def test_grad_repeats_bit_for_bit():
    for m, n, k in ((128, 128, 8192), (700, 1056, 1000), (1304, 1408, 4000)):
        g = torch.randn(m, k, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
        c, s = (t.cuda() for t in R.random_codes(k, n, E4M3, 2))
        first = ops().mx_matmul_grad(g, c, s, m, n, k, 0, False)
        assert all(torch.equal(first, ops().mx_matmul_grad(g, c, s, m, n, k, 0, False)) for _ in range(4))


def test_gradient_rows_beyond_the_result_are_left_alone():
    from mor_b200 import cabi
    for m, n, k in ((5, 64, 40), (133, 160, 70), (300, 96, 4096), (2309, 1312, 100)):
        g = torch.randn(m, (k + 7) // 8 * 8, device="cuda").to(torch.bfloat16)
        c, s = (t.cuda() for t in R.random_codes(k, n, E4M3, 2))
        out = torch.full((m * n + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
        cabi.call("mor_b200_mx_matmul_grad", g.data_ptr(), g.shape[1], c.data_ptr(), s.data_ptr(), m, n, k, 0, 0, out.data_ptr(),
                  torch.cuda.current_stream().cuda_stream)
        assert bool((out[m * n:] == 7.0).all())
        assert torch.equal(out[:m * n].view(m, n), ops().mx_matmul_grad(g[:, :k], c, s, m, n, k, 0, False))


@pytest.mark.parametrize("fmt", [E4M3, E5M2, E2M1])
@pytest.mark.parametrize("m,n,k,across", [(2, 3200, 5488, True), (2, 3200, 5486, True), (2, 3200, 5488, False), (1, 128, 8192, True),
                                          (2304, 1312, 2000, True), (1304, 1408, 4000, False)])
def test_grad_repeats_beside_others(m, n, k, across, fmt):
    """on three streams at once, where the loads of one call are late in any order: a step's codes may land before an
    earlier step's, and a gradient of two rows, nearly all of whose tile lies outside, before either"""
    g = torch.randn((k, m) if across else (m, k), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    c, s = (t.cuda() for t in R.random_codes(k, n, fmt, 2))
    want = check_grad(m, n, k, fmt, across, seed=2, g=g, w=(c.cpu(), s.cpu()))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(30):
        outs = []
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(ops().mx_matmul_grad(g, c, s, m, n, k, fmt, across))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("fmt", [E4M3, E2M1])
@pytest.mark.parametrize("m,n,k", [(1, 3200, 5504), (40, 1000, 4128), (100, 2048, 8192), (1300, 1400, 2080), (2400, 2300, 1024)])
def test_product_repeats_beside_others(m, n, k, fmt):
    a, b, _ = product_case(m, n, k, fmt, fmt, 8, False)
    args = [t.cuda() for t in (*a, *b)]
    want = check_product(m, n, k, fmt, fmt, a=a, b=b)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(30):
        outs = []
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(ops().mx_matmul(*args, m, n, k, fmt, fmt))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


# ------------------------------------------------------------------------------------------------ column sums
@pytest.mark.parametrize("rows,cols", [(0, 40), (1, 1), (1, 64), (3, 8), (31, 65), (33, 7), (127, 72), (128, 64), (141, 232), (513, 1003), (5003, 64),
                                       (4096, 4096), (300, 8192), (70000, 24)])
def test_column_sums(rows, cols):
    g = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16)
    got = ops().column_sums(g.cuda(), rows, cols)
    assert got.shape == (cols,) and got.dtype == torch.bfloat16
    exact, size = g.double().sum(0), g.double().abs().sum(0)
    # one rounding of the result, and half a step of binary32 of what has been added up for each addition
    assert bool(((got.double().cpu() - exact).abs() <= 2.0 ** -8 * exact.abs() + rows * 2.0 ** -24 * size + 2.0 ** -133).all())
    assert torch.equal(got, ops().column_sums(g.cuda(), rows, cols))


def test_column_sums_strides_and_refusals():
    o = ops()
    wide = torch.randn(200, 96, device="cuda").to(torch.bfloat16)
    for v in (wide[:, 8:72], wide[:, 1:64], wide.t(), wide[::2, :40], wide[:1].expand(50, 96), wide[3:4]):
        exact = v.double().sum(0)
        assert bool(((o.column_sums(v, *v.shape).double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 200 * 2.0 ** -24 * v.double().abs().sum(0)).all())
    x = wide.clone()
    x[5, 3], x[6, 4] = float("nan"), float("inf")
    s = o.column_sums(x, 200, 96)
    assert bool(torch.isnan(s[3])) and bool(torch.isinf(s[4])) and bool(torch.isfinite(s[5:]).all())
    for bad in (lambda: o.column_sums(wide.float(), 200, 96), lambda: o.column_sums(wide, 100, 96), lambda: o.column_sums(wide[0], 1, 96)):
        with pytest.raises(RuntimeError):
            bad()


# ------------------------------------------------------------------------------------------------ more than 2^31 elements
def test_quantisation_past_32_bits():
    r, c = 70000, 32768
    x = torch.zeros(r, c, dtype=torch.bfloat16, device="cuda")
    at = [0, 1, r // 2, r - 2, r - 1]
    x[at] = torch.randn(len(at), c, device="cuda").to(torch.bfloat16)
    p, s = ops().quantize_mx_fp4(x, r, c, 32)
    ep, es = R.quantize_fp4(x[at].double().cpu().numpy())
    assert torch.equal(p[at].cpu(), ep) and torch.equal(s[at].cpu(), es)
    del x
    y = ops().dequantize_mx(p, s, r, c, 32, E2M1)
    assert torch.equal(y[at].double().cpu(), R.decode(ep, es, E2M1))
    assert int((y != 0).sum(dtype=torch.int64)) == int((y[at] != 0).sum())


def test_products_past_32_bits():
    m, n, k = 66000, 33000, 32
    a, b = R.random_codes(m, k, E4M3, 1), R.random_codes(n, k, E4M3, 2)
    y = ops().mx_matmul(a[0].cuda(), a[1].cuda(), b[0].cuda(), b[1].cuda(), m, n, k, 0, 0)
    va, vb = R.decode(*a, E4M3).cuda(), R.decode(*b, E4M3).cuda()
    for rows in (slice(0, 3), slice(m - 300, m)):
        exact, size = va[rows] @ vb.t(), va[rows].abs() @ vb.abs().t()
        close(y[rows], exact.cpu(), size.cpu(), k, 32)
    del y, va, vb
    n = 32800                       # the same from a gradient, whose outputs are a multiple of 32 wide
    g = torch.randn(m, 16, device="cuda").to(torch.bfloat16)
    w = R.random_codes(16, n, E2M1, 3)
    y = ops().mx_matmul_grad(g, w[0].cuda(), w[1].cuda(), m, n, 16, E2M1, False)
    gd, wd = g[-300:].double().cpu(), R.decode(*w, E2M1)
    close(y[-300:], gd @ wd, gd.abs() @ wd.abs(), 16, 16)


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    o = ops()
    x = torch.randn(8, 64, device="cuda").to(torch.bfloat16)
    c, s = o.quantize_mx_fp4(x, 8, 64, 32)
    u8 = lambda *sh: torch.zeros(*sh, dtype=torch.uint8, device="cuda")  # noqa: E731
    for bad in (lambda: o.quantize_mx_fp4(x, 8, 64, 16), lambda: o.quantize_mx_fp4(x, 8, 32, 32), lambda: o.quantize_mx_fp4(x.half(), 8, 64, 32),
                lambda: o.quantize_mx_fp4(x[:, :48], 8, 48, 32), lambda: o.quantize_mx_fp4(x[0], 1, 64, 32),
                lambda: o.dequantize_mx(c, s, 8, 64, 32, 2), lambda: o.dequantize_mx(c, s, 8, 64, 32, 0),
                lambda: o.dequantize_mx(c, s, 8, 64, 48, 4), lambda: o.dequantize_mx(c, s, 8, 64, 32, 4, torch.float16),
                lambda: o.dequantize_mx(c, s.cpu(), 8, 64, 32, 4), lambda: o.dequantize_mx(c.float(), s, 8, 64, 32, 4),
                lambda: o.mx_matmul(c, s, c, s, 8, 8, 64, 4, 0), lambda: o.mx_matmul(c, s, c, s, 8, 8, 64, 3, 3),
                lambda: o.mx_matmul(c, s, c, s, 8, 8, 32, 4, 4), lambda: o.mx_matmul(c, s, c, s, 8, 9, 64, 4, 4),
                lambda: o.mx_matmul(u8(8, 0), u8(8, 0), u8(8, 0), u8(8, 0), 8, 8, 0, 4, 4),
                lambda: o.mx_matmul(u8(8, 48), u8(8, 1), u8(8, 48), u8(8, 1), 8, 8, 48, 0, 0),
                lambda: o.mx_matmul(c, s, c, s, 8, 8, 64, 4, 4, torch.zeros(8, device="cuda")),
                lambda: o.mx_matmul(c, s, c, s, 8, 8, 64, 4, 4, torch.zeros(7, device="cuda", dtype=torch.bfloat16)),
                lambda: o.mx_matmul(c, s, c.cpu(), s, 8, 8, 64, 4, 4),
                lambda: o.mx_matmul_grad(x, c, s, 8, 64, 64, 4, False), lambda: o.mx_matmul_grad(x.float(), c, s, 64, 64, 8, 4, True),
                lambda: o.mx_matmul_grad(x, c, s, 64, 64, 8, 2, True), lambda: o.mx_matmul_grad(x, c, s, 64, 48, 8, 4, True),
                lambda: o.mx_matmul_grad(x, c, s, 64, 64, 8, 4, False)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(NotImplementedError):      # CUDA only
        o.quantize_mx_fp4(x.cpu(), 8, 64, 32)
