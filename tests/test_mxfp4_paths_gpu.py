"""GPU tests of the MXFP4 kernels at sizes that reach each of them, against tests/mxfp4_plain.py."""
import pytest

from test_mxfp4_gpu import layer_case, same

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# fused with its quantiser, few rows, exchanged operands, few tiles of a long K, CTAs, CTA pairs
@pytest.mark.parametrize("layer", [(5, 320, 72), (40, 96, 200), (20, 8192, 72), (100, 320, 24), (130, 4096, 72), (1024, 96, 4096),
                                   (2305, 96, 2184)])
def test_relu_gives_zero_for_nan(cb, device, layer):
    """As in the other fused layer: the clip is fmaxf(0, .), which returns its other operand for a NaN."""
    x, (w, sw), bias, sums = layer_case(device, torch.bfloat16, *layer)
    rows = [0, layer[0] - 1]
    x[rows, layer[1] - 1] = float("nan")
    y = cb.linear_mxfp4(x, w, sw, bias)
    clipped = cb.linear_mxfp4(x, w, sw, bias, relu=True)
    cb.check_device()
    assert torch.isnan(y[rows]).all() and int(torch.isnan(y).sum()) == 2 * layer[2]
    want = (sums + bias.double()).clamp(min=0)
    want[rows] = 0
    assert same(clipped, want.bfloat16())
