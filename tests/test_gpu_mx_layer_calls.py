"""Calls of the layer on microscaled operands as programs around it make them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["e4m3", "e2m1"])
def test_a_pass_computes_the_gradients_that_it_is_asked_for(name):
    """the others are neither computed nor given memory; those asked for are the same bits as in a whole pass"""
    from mor_b200.nn import MXLinear
    torch.manual_seed(0)
    layer = MXLinear(2048, 2048, device="cuda", elem_format=name)
    x = torch.randn(2048, 2048, device="cuda").to(torch.bfloat16).requires_grad_()
    leaves = {"x": x, "weight": layer.weight, "bias": layer.bias}
    y = layer(x)
    g = torch.randn_like(y)
    whole = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), g, retain_graph=True)))
    for asked in (("x",), ("weight",), ("bias",), ("x", "bias"), ("weight", "bias"), ("x", "weight")):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = torch.autograd.grad(y, [leaves[a] for a in asked], g, retain_graph=True)
        peak = torch.cuda.max_memory_allocated() - before
        assert all(torch.equal(t, whole[a]) for t, a in zip(got, asked)), asked
        assert peak < sum(whole[a].numel() * 2 for a in asked) + (1 << 20), (asked, peak)
    layer.weight.grad = None
    y.backward(g, inputs=[layer.weight])
    assert torch.equal(layer.weight.grad, whole["weight"]) and x.grad is None and layer.bias.grad is None


@pytest.mark.parametrize("name", ["e4m3", "e2m1"])
@pytest.mark.parametrize("shape", [(64,), (6, 64), (2, 3, 64), (2, 1, 3, 64), (0, 3, 64)])
def test_results_can_be_written_in_place(shape, name):
    """as those of torch's own layer can: an activation in place, a residual added"""
    from mor_b200.nn import MXLinear
    torch.manual_seed(0)
    layer = MXLinear(64, 32, device="cuda", elem_format=name)
    x = torch.randn(*shape, device="cuda").to(torch.bfloat16).requires_grad_()
    r = torch.randn(*shape[:-1], 32, device="cuda").to(torch.bfloat16).requires_grad_()

    def grads(f):
        return torch.autograd.grad(f().float().sum(), (x, r, layer.weight, layer.bias), allow_unused=True)
    for inside, beside in ((lambda: torch.relu_(layer(x)) + r, lambda: torch.relu(layer(x)) + r), (lambda: layer(x).add_(r), lambda: layer(x) + r)):
        assert torch.equal(inside(), beside())
        assert all(torch.equal(u, v) for u, v in zip(grads(inside), grads(beside)))
    packed = layer.pack()
    y = packed(x).add_(r)
    assert y.shape == (*shape[:-1], 32) and torch.equal(y, packed(x) + r) and packed(x).is_contiguous()
    assert torch.equal(torch.autograd.grad(y.float().sum(), r)[0], torch.ones_like(r))


@pytest.mark.parametrize("name", ["e4m3", "e2m1"])
def test_a_packed_layer_may_be_cast_with_the_model_around_it(name):
    """model.float(), model.double() cast its bias, too: the result stays the same bits"""
    from mor_b200.nn import MXLinear
    torch.manual_seed(0)
    packed = MXLinear(64, 40, device="cuda", elem_format=name).pack()
    x = torch.randn(5, 64, device="cuda").to(torch.bfloat16)
    want = packed(x)
    for dtype in (torch.float32, torch.float64, torch.bfloat16):
        packed.to(dtype)
        assert packed.bias.dtype == dtype and torch.equal(packed(x), want)


@pytest.mark.parametrize("name", ["e4m3", "e5m2", "e2m1"])
def test_weights_that_lie_anywhere(name):
    """parameters that are slices of one long tensor, as sharded training has them: the layer takes them, and so does pack()"""
    from mor_b200.nn import MXLinear
    import mor
    torch.manual_seed(0)
    flat = torch.randn(3 + 40 * 64 + 40, device="cuda").to(torch.bfloat16)
    want, layer = (MXLinear(64, 40, device="cuda", elem_format=name) for _ in range(2))
    layer.weight, layer.bias = torch.nn.Parameter(flat[3:-40].view(40, 64)), torch.nn.Parameter(flat[-40:])
    with torch.no_grad():
        want.weight.copy_(layer.weight), want.bias.copy_(layer.bias)
    x = torch.randn(6, 64, device="cuda").to(torch.bfloat16)
    assert layer.weight.data_ptr() % 16 == 6
    assert torch.equal(layer(x), want(x)) and torch.equal(layer.pack()(x), want(x))
    if name != "e2m1":
        for operand in (False, True):
            for u, v in zip(mor.ops.quantize_mx(layer.weight.detach(), 40, 64, 32, 0, operand), mor.ops.quantize_mx(want.weight.detach(), 40, 64, 32, 0, operand)):
                assert torch.equal(u, v)


@pytest.mark.parametrize("name", ["e4m3", "e2m1"])
@pytest.mark.parametrize("shape", [(64,), (5, 64), (2, 3, 64), (0, 64), (2, 0, 64)])
def test_a_layer_of_no_outputs(shape, name):
    from mor_b200.nn import MXLinear
    with pytest.warns(UserWarning, match="zero-element"):
        layer = MXLinear(64, 0, device="cuda", elem_format=name)
    x = torch.randn(*shape, device="cuda").to(torch.bfloat16).requires_grad_()
    y = layer(x)
    y.backward(torch.empty_like(y))
    assert y.shape == (*shape[:-1], 0) and x.grad.shape == x.shape and not bool(x.grad.any())
    assert layer.weight.grad.shape == (0, 64) and layer.bias.grad.shape == (0,) and layer.pack()(x).shape == y.shape
