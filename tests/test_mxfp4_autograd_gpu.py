"""GPU tests of the MXFP4 wrappers beside autograd: they have no derivative, so a call that would drop a gradient is
refused, and one that overwrites values kept for a backward pass is noticed there."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture
def layer(cb, device):
    g = torch.Generator(device=device).manual_seed(8)
    x = torch.randn((4, 64), device=device, generator=g)
    q, s = cb.quantize_mxfp4(torch.randn((24, 64), device=device, generator=g))
    return x, q, s, torch.randn(24, device=device, generator=g)


def test_calls_that_would_drop_a_gradient_are_refused(cb, layer):
    x, q, s, bias = layer
    leaf, tracked_bias = x.clone().requires_grad_(), bias.clone().requires_grad_()
    for out in (torch.empty((24, 64), device=x.device, requires_grad=True), torch.empty((24, 64), device=x.device, requires_grad=True) * 1):
        with pytest.raises(ValueError, match="gradient"):
            cb.dequantize_mxfp4(q, s, 64, torch.float32, out=out)
    y = torch.empty((4, 24), device=x.device, requires_grad=True)
    a, sa = cb.quantize_mxfp4(x)
    for call in (lambda: cb.quantize_mxfp4(leaf), lambda: cb.quantize_mxfp4(leaf * 2, 1), lambda: cb.linear_mxfp4(leaf, q, s),
                 lambda: cb.linear_mxfp4(x, q, s, tracked_bias), lambda: cb.linear_mxfp4(x, q, s, torch.nn.Parameter(bias)),
                 lambda: cb.linear_mxfp4(x, q, s, out=y), lambda: cb.gemm_mxfp4(a, sa, q, s, torch.float32, out=y)):
        with pytest.raises(ValueError, match="gradient"):
            call()


def test_calls_outside_autograd_take_the_same_tensors(cb, layer):
    """Under no_grad and in inference mode, and on detached tensors: what the values alone give."""
    x, q, s, bias = layer
    leaf, tracked_bias = x.clone().requires_grad_(), bias.clone().requires_grad_()
    want = cb.linear_mxfp4(x, q, s, bias)
    codes = cb.quantize_mxfp4(x)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            y = torch.empty((4, 24), device=x.device)
            assert torch.equal(cb.linear_mxfp4(leaf, q, s, tracked_bias), want)
            assert torch.equal(cb.linear_mxfp4(leaf, q, s, tracked_bias, out=y), want) and torch.equal(y, want)
            assert all(torch.equal(a, b) for a, b in zip(cb.quantize_mxfp4(leaf), codes))
    assert torch.equal(cb.linear_mxfp4(leaf.detach(), q, s, tracked_bias.detach()), want)
    cb.check_device()


def test_forward_tangents_are_refused(cb, layer):
    import torch.autograd.forward_ad as fwd

    x, q, s, bias = layer
    with fwd.dual_level():
        dual, dual_bias = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(bias, torch.ones_like(bias))
        for call in (lambda: cb.quantize_mxfp4(dual), lambda: cb.linear_mxfp4(dual, q, s), lambda: cb.linear_mxfp4(x, q, s, dual_bias)):
            with pytest.raises(ValueError, match="gradient"):
                call()


def test_values_kept_for_a_backward_pass_are_not_overwritten_unnoticed(cb, layer):
    x, q, s, _ = layer
    a, sa = cb.quantize_mxfp4(x)
    for shape, write in (((24, 64), lambda o: cb.dequantize_mxfp4(q, s, 64, torch.float32, out=o)),
                         ((4, 24), lambda o: cb.gemm_mxfp4(a, sa, q, s, torch.float32, out=o)),
                         ((4, 24), lambda o: cb.linear_mxfp4(x, q, s, out=o))):
        kept = torch.ones(shape, device=x.device)
        leaf = torch.ones(shape, device=x.device, requires_grad=True)
        loss = (leaf * kept).sum()
        write(kept)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
        loss = (leaf * kept).sum()  # kept anew: nothing has been written since
        loss.backward()
        assert torch.equal(leaf.grad, kept)
    cb.check_device()
