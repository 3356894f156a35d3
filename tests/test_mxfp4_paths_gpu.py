"""GPU tests of the MXFP4 kernels at sizes where each keeps its SMs busy for several rounds, against tests/mxfp4_plain.py:
CTAs and CTA pairs that work through tiles and rings of shared memory, the layer's tail in every kernel, quantisers whose warps
take several steps of a row, and scales at both ends of their range.

Bits are compared wherever every partial sum is a number that fp32 holds (as in test_mxfp4_gpu.py)."""
import pytest

import mxfp4_plain as plain
from test_mxfp4_gpu import DTYPES, check_quantised, exact_case, generator, layer_case, same

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# M, N, K: five tiles a CTA pair and nine k-blocks each (a ring of five stages), C aligned or not; up to three tiles of a CTA
PRODUCTS = [(4600, 4360, 2056), (4609, 4355, 2080), (1024, 4096, 2080), (100, 38096, 1544), (100, 38101, 1544), (20000, 40, 1544)]


@pytest.mark.parametrize("shape", PRODUCTS)
def test_product_of_many_tiles_and_many_blocks_is_exact(cb, device, shape):
    (a, sa), (b, sb), want = exact_case(device, *shape)
    for dtype in DTYPES:
        got = cb.gemm_mxfp4(a, sa, b, sb, dtype)
        cb.check_device()
        assert same(got, want.to(dtype)), dtype


# batch, in, out: CTA pairs with two and five tiles, CTAs with two and three, a split of K, operands that change places
LAYERS = [(2305, 328, 2184), (2048, 96, 11008), (1024, 96, 4096), (100, 160, 38101), (128, 2816, 264), (100, 2048, 24), (1000, 328, 17),
          (5000, 64, 32)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layer", LAYERS)
def test_layers_tail_in_every_kernel(cb, device, layer, dtype):
    x, (w, sw), bias, sums = layer_case(device, dtype, *layer)
    for with_bias in (False, True):
        for relu in (False, True):
            y = cb.linear_mxfp4(x, w, sw, bias if with_bias else None, relu=relu)
            cb.check_device()
            want = sums + bias.double() if with_bias else sums
            want = want.clamp(min=0) if relu else want
            assert same(y, want.to(dtype))


# rows of more than one group of 4096 elements, enough of them that a warp takes a whole group; 16-byte aligned or not
BIG = [(8200, 4104, 4104, 0), (7201, 5003, 5003, 0), (7201, 5003, 5008, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("along", [0, 1])
@pytest.mark.parametrize("rows,cols,pitch,shift", BIG)
def test_quantisers_of_long_rows_there_and_back(cb, device, rows, cols, pitch, shift, along, dtype):
    g = generator(device, rows + cols + shift + along)
    room = torch.randn((rows, pitch), device=device, generator=g)
    room *= torch.exp2(torch.randint(-6, 7, (rows, 1), device=device, generator=g).float())
    x = room.to(dtype)[:, shift : shift + cols]
    q, s = check_quantised(cb, x, along)
    want = plain.values(*plain.unpack(q, s))[:, : rows if along else cols]
    for out in DTYPES:
        q, s = cb.quantize_mxfp4(x, along)  # the way back follows in the stream at once
        assert same(cb.dequantize_mxfp4(q, s, want.shape[1], out), want.to(out))


def test_plain_launches_of_long_rows_give_the_same(cb, device):
    """Grids that are launched ahead of their predecessor's end, and the same launched plainly."""
    from cudaintro_b200 import capi

    x = torch.randn((8200, 4104), device=device, generator=generator(device, 6)).bfloat16()

    def everything():
        out = []
        for _ in range(3):
            for along in (0, 1):
                q, s = cb.quantize_mxfp4(x, along)
                out += [q, s, cb.dequantize_mxfp4(q, s), cb.gemm_mxfp4(q[:4096], s[:32], q[:200], s[:2])]
        return out

    first = everything()
    try:
        capi.lib.b200_set_dependent_launch(0)
        second = everything()
    finally:
        capi.lib.b200_set_dependent_launch(1)
    cb.check_device()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


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


@pytest.mark.parametrize("shape", [(3, 40, 96), (100, 20, 160), (40, 300, 768), (200, 300, 4096), (2304, 2304, 96)])
@pytest.mark.parametrize("low_a,low_b", [(-127, 125), (125, -127), (-100, 0), (0, 100), (-60, -60), (-65, -65)])
def test_scales_at_the_ends_of_their_range(cb, device, shape, low_a, low_b):
    """Block exponents far below and above 0, up to both ends of the scale byte, where the products and sums are still
    numbers that fp32 holds: powers of two times the exact case (products 2^(low_a + low_b) .. 2^4 times that)."""
    M, N, K = shape
    g = generator(device, M + N + K)
    high = 2 if max(low_a, low_b) < 126 else 0
    a, b = plain.random_packed(M, K, low_a, min(low_a + high, 127), g), plain.random_packed(N, K, low_b, min(low_b + high, 127), g)
    (qa, sa), (qb, sb) = plain.pack(*a), plain.pack(*b)
    want = plain.values(*a) @ plain.values(*b).t()
    got = cb.gemm_mxfp4(qa, sa, qb, sb, torch.float32)
    cb.check_device()
    assert same(got, want.float())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layer", [(1, 31, 40), (3, 1031, 72), (16, 77, 264), (5, 4099, 136), (16, 11007, 96), (32, 333, 40)])
def test_small_layers_take_rows_of_any_length_and_views(cb, device, layer, dtype):
    """Rows that the product quantises itself, aligned to their elements only; x, bias and out begin inside larger tensors,
    and what lies around the result stays."""
    batch, in_f, out_f = layer
    x, (w, sw), bias, sums = layer_case(device, dtype, *layer)
    if in_f > 7281:  # beyond that fp32 holds the sums only of fewer terms
        w[:, 2048:] = 0
        sums = x[:, :4096].double() @ plain.values(*plain.unpack(w, sw))[:, :4096].t()
    x_room = torch.full((batch * in_f + 3,), float("nan"), dtype=dtype, device=device)
    bias_room = torch.full((out_f + 1,), float("nan"), device=device)
    out_room = torch.full((batch * out_f + 2,), 77.0, dtype=dtype, device=device)
    x_view, bias_view, out = x_room[1:-2].view(batch, in_f), bias_room[1:], out_room[1:-1].view(batch, out_f)
    x_view.copy_(x)
    bias_view.copy_(bias)
    assert cb.linear_mxfp4(x_view, w, sw, bias_view, out=out).data_ptr() == out.data_ptr()
    cb.check_device()
    want = (sums + bias.double()).to(dtype)
    assert same(out, want) and (out_room[[0, -1]] == 77).all()
    assert same(cb.linear_mxfp4(x, w, sw, bias), want)


@pytest.mark.parametrize("layer", [(1, 4096, 1032), (16, 4104, 520), (32, 4096, 136), (3, 96, 18944)])
def test_a_lost_arrival_in_a_small_layer_is_reported(cb, device, layer):
    """The kernel that quantises its rows gives up its waits too, and the next call is right."""
    from cudaintro_b200 import capi

    x, w, bias, sums = layer_case(device, torch.bfloat16, *layer)
    want = (sums + bias.double()).bfloat16()
    assert same(cb.linear_mxfp4(x, *w, bias), want)
    cb.check_device()
    try:
        capi._check(capi.lib.b200_test_lose_arrival(0, 50_000_000))
        cb.linear_mxfp4(x, *w, bias)
        with pytest.raises(cb.B200Error) as info:
            cb.check_device()
        assert info.value.status == 4
    finally:
        capi._check(capi.lib.b200_test_lose_arrival(-1, 0))
    for _ in range(2):
        assert same(cb.linear_mxfp4(x, *w, bias), want)
    cb.check_device()


def test_layers_with_workspaces_in_two_graphs_at_once(cb, device):
    """Layers whose rows are quantised in a launch of their own, captured twice and replayed at the same time on two
    streams while eager calls run on a third: every one has a workspace to itself."""
    shapes = [(300, 1024, 520), (2305, 96, 2184), (40, 8192, 72)]
    cases = [layer_case(device, torch.bfloat16, *s) for s in shapes]
    exact = [(sums + bias.double()).bfloat16() if s[1] <= 7281 else None for s, (_, _, bias, sums) in zip(shapes, cases)]

    def step():
        return [cb.linear_mxfp4(x, *w, bias) for x, w, bias, _ in cases]

    alone = step()
    torch.cuda.synchronize()
    assert all(want is None or same(y, want) for y, want in zip(alone, exact))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step() + step())
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = step()
    torch.cuda.synchronize()
    cb.check_device()
    for ys in (outs[0][:3], outs[0][3:], outs[1][:3], outs[1][3:], eager):
        assert all(torch.equal(y, want) for y, want in zip(ys, alone))
