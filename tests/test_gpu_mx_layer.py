"""The microscaled operators used together: a linear layer's training step and its serving form."""
import math

import pytest
import torch

import mx_reference as R
from test_gpu_mx import STEP, close

pytestmark = pytest.mark.gpu
FORMATS = {"e4m3": 0, "e5m2": 1, "e2m1": 4}


def quantised(x2, name):
    """float64 values that the layer's quantiser gives for a [rows, cols] tensor, by the definition"""
    f = FORMATS[name]
    x = x2.detach().double().cpu()
    if f == 4:
        return R.decode(*R.quantize_fp4(x.numpy()), f)
    top, frac = (8, 1.75) if f == 0 else (15, 1.75)
    amax = x.reshape(x.shape[0], -1, 32).abs().amax(2)
    m, e = torch.frexp(amax)
    up = torch.where(amax > 0, top - (e - 1) - (2 * m > frac).to(e.dtype), 0).double()
    k = (2.0 ** up).repeat_interleave(32, 1)
    q = (x * k).float().to(torch.float8_e4m3fn if f == 0 else torch.float8_e5m2).double()
    return q / k


def make(name, shape, n, seed=0, dtype=torch.bfloat16, bias=True):
    from mor_b200.nn import MXLinear
    torch.manual_seed(seed)
    layer = MXLinear(shape[-1], n, bias=bias, device="cuda", dtype=dtype, elem_format=name)
    x = torch.randn(*shape, device="cuda", dtype=dtype, requires_grad=True)
    g = torch.randn(*shape[:-1], n, device="cuda").to(torch.bfloat16)
    return layer, x, g


@pytest.mark.parametrize("name", ["e4m3", "e5m2", "e2m1"])
@pytest.mark.parametrize("shape,n", [((4, 64, 512), 256), ((300, 96), 72), ((1, 32), 8), ((3, 5, 160), 33), ((2048,), 64), ((1024, 1024), 1024)])
def test_step_against_the_formula(name, shape, n):
    layer, x, g = make(name, shape, n)
    if len(shape) == 1:
        g = g.reshape(n)
    y = layer(x)
    assert y.shape == (*shape[:-1], n) and y.dtype == torch.bfloat16
    y.backward(g)
    k = shape[-1]
    xq, wq = quantised(x.reshape(-1, k), name), quantised(layer.weight, name)
    gd, b = g.reshape(-1, n).double().cpu(), layer.bias.detach().double().cpu()
    m = xq.shape[0]
    close(y.reshape(m, n), xq @ wq.t() + b, xq.abs() @ wq.abs().t() + b.abs(), k, STEP[FORMATS[name]])
    close(x.grad.reshape(m, k), gd @ wq, gd.abs() @ wq.abs(), n, 16)
    close(layer.weight.grad, gd.t() @ xq, gd.abs().t() @ xq.abs(), m, 16)
    close(layer.bias.grad, gd.sum(0), gd.abs().sum(0), m, 1)
    assert x.grad.dtype == x.dtype and layer.weight.grad.shape == layer.weight.shape


@pytest.mark.parametrize("name", ["e4m3", "e2m1"])
def test_gradient_against_differences(name):
    """Inputs on the quantiser's grid move by whole codes, so y is linear between them: <g, y(x + d) - y(x)> = <dx, d>."""
    from mor_b200.nn import mx_linear
    m, n, k = 48, 64, 96
    gen = torch.Generator().manual_seed(1)
    x = torch.randint(-3, 4, (m, k), generator=gen).float()
    w = torch.randint(-3, 4, (n, k), generator=gen).float()
    x[:, ::32], w[:, ::32] = 4.0, 4.0                 # fixes every group's scale
    dx, dw = torch.zeros(m, k), torch.zeros(n, k)
    dx[:, 1::32], dw[:, 5::32] = 1.0, -1.0            # whole numbers up to 4 are codes of both formats under these scales
    g = torch.randint(-2, 3, (m, n), generator=gen).float()
    x, w, dx, dw, g = (t.to(torch.bfloat16).cuda() for t in (x, w, dx, dw, g))
    x.requires_grad_(), w.requires_grad_()
    f = FORMATS[name]
    y = mx_linear(x, w, None, f)
    gx, gw = torch.autograd.grad(y, (x, w), g)

    def inner(u, v):
        return float((u.double() * v.double()).sum())
    with torch.no_grad():
        # y holds whole numbers below 2^11; those a bf16 cannot hold are rounded by at most half a step
        for moved, want in ((mx_linear(x + dx, w, None, f), inner(gx, dx)), (mx_linear(x, w + dw, None, f), inner(gw, dw))):
            slack = float((g.abs().double() * (moved.abs().double() + y.abs().double())).sum()) * 2.0 ** -8
            slack += float((gx.abs().double() * dx.abs().double()).sum() + (gw.abs().double() * dw.abs().double()).sum()) * 2.0 ** -8
            assert abs(inner(g, moved.double() - y.double()) - want) <= slack


def test_float32_layer_and_partial_gradients():
    layer, x, g = make("e2m1", (40, 64), 24, dtype=torch.float32)
    y = layer(x)
    gx, = torch.autograd.grad(y, x, g)
    assert gx.dtype == torch.float32
    layer.weight.requires_grad_(False)
    x2 = x.detach().requires_grad_()
    gx2, gb = torch.autograd.grad(layer(x2), (x2, layer.bias), g)
    assert torch.equal(gx, gx2) and gb.dtype == torch.float32
    x3 = x.detach()
    layer.weight.requires_grad_(True)
    gw, = torch.autograd.grad(layer(x3), layer.weight, g)
    assert gw.dtype == torch.float32 and gw.shape == layer.weight.shape
    strided = torch.randn(64, 80, device="cuda").t()[:40]     # not contiguous, gradient an expanded scalar
    strided = strided[:, :64]
    layer(strided).sum().backward()
    assert torch.isfinite(layer.weight.grad).all()


@pytest.mark.parametrize("fmt", [0, 1, 3])
@pytest.mark.parametrize("rows,cols,by", [(1, 32, 32), (3, 32, 32), (1, 8, 8), (5, 96, 32), (129, 32, 16), (141, 64, 64), (67, 4128, 32), (1000, 40, 8)])
def test_eight_bit_quantisation_of_any_number_of_rows(rows, cols, by, fmt):
    """sizes that are no multiple of 256 elements, against the CPU oracle, and nothing written behind them"""
    import oracle
    from mor_b200 import cabi
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16)
    codes, scales = oracle.quantize_mx(oracle.bf16_bits(x), by, fmt)
    d = x.cuda()
    p = torch.full((rows * cols + 512,), 9, dtype=torch.uint8, device="cuda")
    s = torch.full((rows * cols // by + 512,), 9, dtype=torch.uint8, device="cuda")
    cabi.call("mor_b200_quantize_mx", d.data_ptr(), p.data_ptr(), s.data_ptr(), rows, cols, by, fmt, torch.cuda.current_stream().cuda_stream)
    assert (p[:rows * cols].cpu().numpy() == codes.reshape(-1)).all() and (s[:rows * cols // by].cpu().numpy() == scales.reshape(-1)).all()
    assert bool((p[rows * cols:] == 9).all()) and bool((s[rows * cols // by:] == 9).all())
    if fmt == 3:
        p6 = torch.full((rows * cols * 3 // 4 + 512,), 9, dtype=torch.uint8, device="cuda")
        cabi.call("mor_b200_quantize_mx_fp6", d.data_ptr(), p6.data_ptr(), s.data_ptr(), rows, cols, by, torch.cuda.current_stream().cuda_stream)
        assert (p6[:rows * cols * 3 // 4].cpu().numpy() == oracle.pack_fp6(codes).reshape(-1)).all() and bool((p6[rows * cols * 3 // 4:] == 9).all())


@pytest.mark.parametrize("name", ["e4m3", "e2m1"])
def test_no_tokens(name):
    layer, x, g = make(name, (0, 64), 40)
    y = layer(x)
    y.backward(g)
    assert y.shape == (0, 40) and x.grad.shape == (0, 64)
    assert not bool(layer.weight.grad.any()) and not bool(layer.bias.grad.any())
    assert layer.pack()(x).shape == (0, 40)


@pytest.mark.parametrize("name", ["e4m3", "e2m1"])
def test_what_is_kept_is_the_codes(name):
    layer, x, g = make(name, (256, 512), 128, bias=False)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        layer(x)
    assert all(t.dtype == torch.uint8 for t in kept)
    bits = 8 if name == "e4m3" else 4
    assert sum(t.numel() for t in kept) == (256 + 128) * 512 * bits // 8 + (256 + 128) * 16


@pytest.mark.parametrize("name", ["e4m3", "e2m1"])
@pytest.mark.parametrize("tokens", [1, 3, 70])
def test_packed_layer_gives_the_same_bits(name, tokens):
    layer, x, _ = make(name, (tokens, 512), 1000)
    packed = layer.pack()
    y = packed(x)
    assert torch.equal(y, layer(x).detach()) and not y.requires_grad
    assert torch.equal(packed(x[None, :, None]), y[None, :, None])
    with pytest.raises(RuntimeError, match="must be"):
        packed(x[:, :64])
    assert not list(packed.parameters()) and "payload" in packed.state_dict()
    with torch.no_grad():
        layer.weight.zero_()
    assert bool(packed(x).any())          # its weights are its own


def test_captured_step_replays_with_new_values():
    from mor_b200.nn import mx_linear
    torch.manual_seed(3)
    x = torch.randn(200, 256, device="cuda").to(torch.bfloat16).requires_grad_()
    w = torch.randn(128, 256, device="cuda").to(torch.bfloat16).requires_grad_()
    b = torch.randn(128, device="cuda").to(torch.bfloat16).requires_grad_()
    g = torch.randn(200, 128, device="cuda").to(torch.bfloat16)

    def step():
        outs = []
        for f in (0, 4):
            y = mx_linear(x, w, b, f)
            outs += [y.detach(), *torch.autograd.grad(y, (x, w, b), g)]
        return outs
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        outs2 = step()
    with torch.no_grad():
        x.copy_(torch.randn(200, 256)), w.copy_(torch.randn(128, 256)), g.copy_(torch.randn(200, 128))
    graph.replay()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):         # two captured graphs at once share nothing
        second.replay()
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    assert all(torch.equal(u, v) for u, v in zip(outs, want)) and all(torch.equal(u, v) for u, v in zip(outs2, want))


def test_gradients_have_no_gradient():
    from mor_b200.nn import mx_linear
    x = torch.randn(8, 32, device="cuda").to(torch.bfloat16).requires_grad_()
    w = torch.randn(8, 32, device="cuda").to(torch.bfloat16).requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(mx_linear(x, w).float().square().sum(), x, create_graph=True)
    with torch.no_grad():
        assert not mx_linear(x, w).requires_grad


def test_layer_refusals():
    from mor_b200.nn import mx_linear
    x = torch.randn(8, 32, device="cuda").to(torch.bfloat16)
    with pytest.raises(ValueError):
        mx_linear(x, x[:, :16])
    with pytest.raises(RuntimeError, match="one device"):
        mx_linear(x, x.cpu())
    with pytest.raises(RuntimeError, match="bfloat16"):
        mx_linear(x.float(), x, None, 0)             # the 8-bit quantiser takes bfloat16
    with pytest.raises(RuntimeError, match="multiple of 32"):
        mx_linear(x[:, :24].contiguous(), x[:, :24].contiguous(), None, 4)
    with pytest.raises(RuntimeError, match="bias"):
        mx_linear(x, x, torch.zeros(3, device="cuda", dtype=torch.bfloat16), 4)


def test_training_runs():
    from mor_b200.nn import MXLinear
    torch.manual_seed(0)
    net = torch.nn.Sequential(MXLinear(64, 96, device="cuda", elem_format="e4m3"), torch.nn.ReLU(),
                              MXLinear(96, 32, device="cuda", elem_format="e2m1"))
    opt = torch.optim.SGD(net.parameters(), lr=0.01)
    x = torch.randn(50, 64, device="cuda").to(torch.bfloat16)
    for _ in range(3):
        opt.zero_grad()
        loss = net(x).float().square().mean()
        loss.backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in net.parameters())
        opt.step()
    assert math.isfinite(loss.item())
