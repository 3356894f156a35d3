"""GPU tests of the MXFP4 operators (quantise, dequantise, product, linear layer) against tests/mxfp4_plain.py.

Quantisation and dequantisation are compared bit for bit.  Products are compared bit for bit where every partial
sum is a number that fp32 holds (block exponents within -1..1 and K <= 7281: products are multiples of 2^-4 below
144, so sums stay below 2^24 of those), and within `sum_bound` elsewhere."""
import pytest

import mxfp4_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def generator(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def same(got, want):
    """Equal values, NaN in the same places."""
    got, want = got.double(), want.double()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def check_quantised(cb, x, along):
    q, s = cb.quantize_mxfp4(x, along)
    rows = x.t() if along else x
    code, byte = plain.quantize(rows)
    want_q, want_s = plain.pack(code, byte)
    assert torch.equal(s, want_s)  # the bytes that fill up a tile among them
    assert torch.equal(q, want_q)
    return q, s


# ------------------------------------------------------------------ quantise, dequantise

SHAPES = [(1, 1), (1, 32), (2, 31), (3, 33), (1, 4096), (33, 784), (128, 128), (129, 130), (127, 1001), (257, 513), (640, 96), (300, 2056)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("along", [0, 1])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantise_gives_the_formats_bits(cb, device, shape, along, dtype):
    g = generator(device, shape[0] * 7 + shape[1] + along)
    x = torch.randn(shape, device=device, generator=g) * torch.exp2(torch.randint(-6, 7, shape, device=device, generator=g).float())
    x = x.to(dtype)
    q, s = check_quantised(cb, x, along)
    rows = x.t() if along else x
    want = plain.values(*plain.quantize(rows))[:, : rows.shape[1]]
    for out in DTYPES:
        assert same(cb.dequantize_mxfp4(q, s, rows.shape[1], out), want.to(out))


@pytest.mark.parametrize("along", [0, 1])
def test_quantise_borders_and_special_values(cb, device, along):
    """Every halfway point, the largest magnitudes, zeros of both signs, subnormals, blocks that are not finite."""
    grid = [0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0, 7.9990234375]
    line = torch.zeros(32, dtype=torch.float64)
    line[: len(grid)] = torch.tensor(grid, dtype=torch.float64)
    eps = torch.zeros(32, dtype=torch.float64)
    eps[: len(grid)] = torch.tensor(grid, dtype=torch.float64) * (1 - 2.0**-20)
    eps[31] = 4.0
    top = torch.finfo(torch.float32).max
    blocks = [line, -line, eps, line * 2.0**-100, line * 2.0**120, line * 2.0**-140, line * 2.0**-149,
              torch.zeros(32, dtype=torch.float64), -torch.zeros(32, dtype=torch.float64),
              torch.full((32,), top, dtype=torch.float64), torch.full((32,), 2.0**-149, dtype=torch.float64)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        b = line.clone()
        b[5] = bad
        blocks.append(b)
    blocks.append(torch.where(torch.arange(32) < 31, 2.0**-149, 2.0**-126).double())
    x = torch.cat(blocks).float().to(device).unsqueeze(0).repeat(3, 1)
    x[1] = x[1].roll(32)
    x = x.t().contiguous() if along else x
    q, s = check_quantised(cb, x, along)
    back = cb.dequantize_mxfp4(q, s, x.shape[1 - along], torch.float32)
    assert same(back, plain.values(*plain.quantize(x.t() if along else x)).float())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("along", [0, 1])
def test_quantise_every_16_bit_value(cb, device, along, dtype):
    """All bit patterns, in order (blocks of one sign and exponent) and shuffled: subnormals, infinities and NaN too."""
    bits = torch.arange(-32768, 32768, device=device).to(torch.int16)
    shuffled = bits[torch.randperm(65536, device=device, generator=generator(device, 4))]
    for b in (bits, shuffled):
        x = b.view(dtype).reshape(256, 256)
        check_quantised(cb, x.t().contiguous() if along else x, along)
    finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    check_quantised(cb, finite, along)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("along", [0, 1])
def test_quantise_takes_strided_and_unaligned_rows(cb, device, along, dtype):
    g = generator(device, 3)
    wide = torch.randn((70, 301), device=device, generator=g).to(dtype)
    for view in (wide[:, :256], wide[:, 1:290], wide[::2, 3:100], wide[5:6, 7:], wide[:, 4:5]):
        check_quantised(cb, view, along)
    aligned = torch.randn((70, 320), device=device, generator=g).to(dtype)
    check_quantised(cb, aligned[:, 64:256], along)


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantise_reads_every_code_and_scale(cb, device, dtype):
    """All codes under all scale bytes, 0 and 255 among them; what lies beyond column K and around the matrix stays."""
    code = torch.arange(16, device=device).repeat(256, 2)
    byte = torch.arange(256, device=device).reshape(256, 1)
    q, s = plain.pack(code, byte)
    want = plain.values(code, byte)
    assert same(cb.dequantize_mxfp4(q, s, 32, dtype), want.to(dtype))
    from cudaintro_b200 import capi

    for K in (1, 7, 8, 31):
        for ldx in (K, 40, 41):
            x = torch.full((258, ldx), 77.0, dtype=dtype, device=device)
            rc = capi.lib.b200_dequantize_mxfp4(capi._code(dtype), q.data_ptr(), s.data_ptr(), x[1].data_ptr(), 256, K, ldx,
                                                torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            assert same(x[1:257, :K], want[:, :K].to(dtype))
            assert (x[0] == 77).all() and (x[257] == 77).all() and (x[:, K:] == 77).all()


# ------------------------------------------------------------------ products

PRODUCTS = [(1, 1, 1), (1, 8, 32), (3, 5, 31), (2, 129, 33), (1, 1000, 4096), (8, 264, 2048), (16, 1000, 7200), (17, 640, 96),
            (32, 4096, 512), (33, 70, 4100), (64, 200, 1024), (65, 384, 640), (100, 136, 784), (128, 128, 128), (129, 127, 65),
            (192, 513, 1000), (256, 192, 96), (257, 512, 784), (256, 256, 256), (512, 520, 7264), (513, 1100, 260),
            (1000, 1544, 2056), (2304, 2176, 320), (4096, 1024, 64), (391, 1037, 160), (515, 333, 96), (2305, 2179, 70), (700, 8, 96),
            (1000, 32, 2056), (4100, 1, 1000), (130, 17, 7000), (33, 32, 4096), (65, 384, 3000), (300, 500, 4097), (128, 4096, 2816),
            (200, 131, 7200), (700, 900, 2304), (100, 33, 6000)]


def exact_case(device, M, N, K):
    g = generator(device, M * 31 + N * 7 + K)
    a, b = plain.random_packed(M, K, -1, 1, g), plain.random_packed(N, K, -1, 1, g)
    return plain.pack(*a), plain.pack(*b), plain.values(*a) @ plain.values(*b).t()


@pytest.mark.parametrize("shape", PRODUCTS)
def test_product_is_exact_where_fp32_holds_the_sums(cb, device, shape):
    (a, sa), (b, sb), want = exact_case(device, *shape)
    for dtype in DTYPES:
        got = cb.gemm_mxfp4(a, sa, b, sb, dtype)
        cb.check_device()
        assert same(got, want.to(dtype)), dtype


@pytest.mark.parametrize("shape", [(1, 520, 4096), (16, 4096, 11008), (40, 72, 333), (300, 264, 8192), (1030, 1100, 2080)])
def test_product_of_wide_ranges_stays_within_the_bound(cb, device, shape):
    M, N, K = shape
    g = generator(device, sum(shape))
    a, b = plain.random_packed(M, K, -30, 10, g), plain.random_packed(N, K, -12, 12, g)
    (qa, sa), (qb, sb) = plain.pack(*a), plain.pack(*b)
    va, vb = plain.values(*a), plain.values(*b)
    for dtype in (torch.float32, torch.bfloat16):
        want, bound = plain.sum_bound(va, vb, dtype)
        got = cb.gemm_mxfp4(qa, sa, qb, sb, dtype)
        cb.check_device()
        assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("shape", [(5, 40, 96), (200, 300, 320)])
def test_nan_blocks_reach_their_rows_and_columns_only(cb, device, shape):
    M, N, K = shape
    g = generator(device, 11)
    a, b = plain.random_packed(M, K, -1, 1, g), plain.random_packed(N, K, -1, 1, g)
    a[1][3, 1] = 255
    b[1][N - 1, 0] = 255
    (qa, sa), (qb, sb) = plain.pack(*a), plain.pack(*b)
    got = cb.gemm_mxfp4(qa, sa, qb, sb, torch.float32)
    cb.check_device()
    want = plain.values(*a) @ plain.values(*b).t()
    assert torch.isnan(want[3]).all() and torch.isnan(want[:, N - 1]).all() and int(torch.isnan(want).sum()) == M + N - 1
    assert same(got, want)


@pytest.mark.parametrize("shape", [(3, 40, 96), (130, 70, 64), (300, 520, 256)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_product_writes_its_own_elements_only(cb, device, shape, dtype):
    """A leading dimension wider than the row, aligned for vector stores or not; what lies around C stays."""
    from cudaintro_b200 import capi

    M, N, K = shape
    (a, sa), (b, sb), want = exact_case(device, M, N, K)
    for ldc, shift in ((N, 0), (N + 8, 0), (N + 3, 0), (N + 8, 1)):
        room = torch.full(((M + 2) * ldc + shift,), 77.0, dtype=dtype, device=device)
        c = room[shift:].view(M + 2, ldc)
        rc = capi.lib.b200_gemm_mxfp4(capi._code(dtype), a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(),
                                      c[1].data_ptr(), M, N, K, ldc, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, capi.lib.b200_last_error()
        cb.check_device()
        assert same(c[1 : M + 1, :N], want.to(dtype))
        assert (c[0] == 77).all() and (c[M + 1] == 77).all() and (c[:, N:] == 77).all() and (room[:shift] == 77).all()


# ------------------------------------------------------------------ linear layer


def layer_case(device, dtype, batch, in_f, out_f):
    """A layer whose sums fp32 holds: activations are elements of the format times 2^-1..2^1, one 6 in each block so
    that the block exponent is known."""
    g = generator(device, batch + in_f + out_f)
    blocks = -(-in_f // 32)
    code, byte = plain.random_packed(batch, in_f, -1, 1, g)
    code[:, 0::32] = 7
    x = plain.values(code, byte)[:, :in_f].to(dtype)
    w = plain.random_packed(out_f, in_f, -1, 1, g)
    bias = torch.randint(-64, 65, (out_f,), device=device, generator=g).float() / 16
    assert blocks * 32 >= in_f
    return x, plain.pack(*w), bias, x.double() @ plain.values(*w)[:, :in_f].t()


LAYERS = [(1, 32, 8), (1, 4096, 1032), (2, 784, 512), (7, 2048, 1024), (16, 4104, 520), (33, 1000, 264), (100, 2048, 1024),
          (128, 96, 256), (257, 784, 512), (520, 1032, 264), (3, 96, 18944), (1, 64, 19000), (32, 4096, 136)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layer", LAYERS)
def test_layer_quantises_multiplies_adds_and_clips(cb, device, layer, dtype):
    x, (w, sw), bias, sums = layer_case(device, dtype, *layer)
    for with_bias in (False, True):
        for relu in (False, True):
            y = cb.linear_mxfp4(x, w, sw, bias if with_bias else None, relu=relu)
            cb.check_device()
            want = sums + bias.double() if with_bias else sums
            want = want.clamp(min=0) if relu else want
            assert same(y, want.to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layer", [(1, 784, 512), (19, 2048, 1024), (300, 1031, 200)])
def test_layer_equals_quantiser_then_product(cb, device, layer, dtype):
    """Ordinary values: the layer against its two halves, and against 64 bits within the bound."""
    batch, in_f, out_f = layer
    g = generator(device, 5)
    x = torch.randn((batch, in_f), device=device, generator=g).to(dtype)
    w, sw = cb.quantize_mxfp4(torch.randn((out_f, in_f), device=device, generator=g) * 0.05)
    y = cb.linear_mxfp4(x, w, sw)
    vx = plain.values(*plain.quantize(x))
    want, bound = plain.sum_bound(vx, plain.values(*plain.unpack(w, sw)), dtype)
    assert ((y.double() - want).abs() <= bound).all()
    q, s = cb.quantize_mxfp4(x)
    parts = cb.gemm_mxfp4(q, s, w, sw, dtype)
    assert ((parts.double() - want).abs() <= bound).all()
    cb.check_device()


def test_layer_keeps_nan_rows_to_themselves(cb, device):
    x, (w, sw), bias, sums = layer_case(device, torch.bfloat16, 5, 320, 72)
    x[2, 100] = float("inf")
    x[4, 319] = float("nan")
    y = cb.linear_mxfp4(x, w, sw, bias)
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all()
    keep = [0, 1, 3]
    assert same(y[keep], (sums + bias.double())[keep].bfloat16())
    cb.check_device()


# ------------------------------------------------------------------ as they are used together


def test_a_training_step_of_a_layer_in_four_bits(cb, device):
    """Forward, input gradient and weight gradient of a layer: three products of operands quantised along the
    dimension that each sums over, from the two directions of the quantiser."""
    g = generator(device, 9)
    batch, in_f, out_f = 96, 160, 224
    x = torch.randn((batch, in_f), device=device, generator=g)
    w = torch.randn((out_f, in_f), device=device, generator=g) * 0.1
    dy = torch.randn((batch, out_f), device=device, generator=g)

    def fake(t, along):  # values of the quantised tensor, in the shape of t
        v = plain.values(*plain.quantize(t.t() if along else t))[:, : t.shape[1 - along]]
        return v.t() if along else v

    y = cb.linear_mxfp4(x, *cb.quantize_mxfp4(w))
    dx = cb.gemm_mxfp4(*cb.quantize_mxfp4(dy), *cb.quantize_mxfp4(w, 1), torch.float32)
    dw = cb.gemm_mxfp4(*cb.quantize_mxfp4(dy, 1), *cb.quantize_mxfp4(x, 1), torch.float32)
    cb.check_device()
    for got, left, right in ((y, fake(x, 0), fake(w, 0).t()), (dx, fake(dy, 0), fake(w, 1)), (dw, fake(dy, 1).t(), fake(x, 1))):
        want, bound = plain.sum_bound(left, right.t(), torch.float32)
        assert got.shape == want.shape and ((got.double() - want).abs() <= bound).all()
    # against differences of the loss sum(dy * y): the products are linear in the operand that is moved, so a step
    # of the exact loss along a direction equals the gradient's product with it
    d = torch.randn((batch, in_f), device=device, generator=g).double()
    loss = lambda t: ((t @ fake(w, 1).t()) * fake(dy, 0)).sum()  # noqa: E731
    step = loss(x.double() + d) - loss(x.double() - d)
    slack = (plain.sum_bound(fake(dy, 0), fake(w, 1).t(), torch.float32)[1] * d.abs()).sum()
    assert (step / 2 - (dx.double() * d).sum()).abs() <= slack + 1e-9 * step.abs()


def test_two_layers_captured_in_a_graph_follow_their_inputs(cb, device):
    """Quantise, product and layer replayed on new inputs, on a stream of their own, equal eager calls."""
    g = generator(device, 21)
    w1 = cb.quantize_mxfp4(torch.randn((512, 256), device=device, generator=g) * 0.1)
    w2 = cb.quantize_mxfp4(torch.randn((96, 512), device=device, generator=g) * 0.1)
    bias = torch.randn(512, device=device, generator=g)
    x = torch.randn((24, 256), device=device, generator=g).bfloat16()

    def step():
        h = cb.linear_mxfp4(x, *w1, bias, relu=True)
        q, s = cb.quantize_mxfp4(h)
        return cb.gemm_mxfp4(q, s, *w2, torch.float32), cb.dequantize_mxfp4(q, s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):
        out2 = step()
    for seed in (1, 2):
        x.copy_(torch.randn((24, 256), device=device, generator=generator(device, seed)))
        graph.replay()
        other.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b, c in zip(out, out2, want):
            assert torch.equal(a, c) and torch.equal(b, c)
    cb.check_device()


def test_calls_on_two_streams_at_once(cb, device):
    """Layers and products in flight together on two streams give what they give alone."""
    cases = [layer_case(device, torch.bfloat16, b, 2048, 1024) for b in (4, 300)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (st, (x, (w, sw), bias, _)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(st):
                got[i].append(cb.linear_mxfp4(x, w, sw, bias))
    torch.cuda.synchronize()
    cb.check_device()
    for ys, (_, _, bias, sums) in zip(got, cases):
        want = (sums + bias.double()).bfloat16()
        assert all(same(y, want) for y in ys)


# ------------------------------------------------------------------ refusals


def test_wrappers_refuse_what_does_not_belong_together(cb, device):
    x = torch.zeros((4, 64), device=device)
    q, s = cb.quantize_mxfp4(x)
    bad = [lambda: cb.quantize_mxfp4(x.double()), lambda: cb.quantize_mxfp4(x.cpu()), lambda: cb.quantize_mxfp4(x, 2),
           lambda: cb.quantize_mxfp4(x.t()), lambda: cb.quantize_mxfp4(x[0]), lambda: cb.quantize_mxfp4(x[:0]),
           lambda: cb.quantize_mxfp4(x[:1].expand(4, 64)),
           lambda: cb.dequantize_mxfp4(q, s, 32), lambda: cb.dequantize_mxfp4(q, s, 65),
           lambda: cb.dequantize_mxfp4(q, s[..., :2], 64), lambda: cb.dequantize_mxfp4(q[:, :8], s, 16),
           lambda: cb.dequantize_mxfp4(q, s, 64, torch.float64),
           lambda: cb.gemm_mxfp4(q, s, q[:, :16].contiguous(), s), lambda: cb.gemm_mxfp4(q, s, q, s, torch.int32),
           lambda: cb.gemm_mxfp4(q, s, q, s.cpu()), lambda: cb.gemm_mxfp4(q, s, q, s, out=torch.empty(4, 5, device=device)),
           lambda: cb.linear_mxfp4(x[:, :32].contiguous(), q, s), lambda: cb.linear_mxfp4(x, q, s, torch.zeros(5, device=device)),
           lambda: cb.linear_mxfp4(x, q, s, torch.zeros(4, device=device).half()), lambda: cb.linear_mxfp4(x.t(), q, s),
           lambda: cb.linear_mxfp4(x, q, s, out=torch.empty(4, 4, device=device).half())]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_what_is_no_tensor_is_refused(cb, device):
    x = torch.zeros((4, 64), device=device)
    q, s = cb.quantize_mxfp4(x)
    for other in (None, 3, [1, 2], "q"):
        for call in (lambda: cb.quantize_mxfp4(other), lambda: cb.dequantize_mxfp4(other, s), lambda: cb.dequantize_mxfp4(q, other),
                     lambda: cb.gemm_mxfp4(q, s, q, other), lambda: cb.gemm_mxfp4(q, other, q, s),
                     lambda: cb.linear_mxfp4(other, q, s), lambda: cb.linear_mxfp4(x, q, other)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: cb.linear_mxfp4(x, q, s, bias=3), lambda: cb.linear_mxfp4(x, q, s, out=3),
                 lambda: cb.dequantize_mxfp4(q, s, dtype=3)):
        with pytest.raises(ValueError):
            call()


def test_values_that_torch_negates_later_are_refused(cb, device):
    x = torch._neg_view(torch.ones((64, 64), device=device))
    q, s = cb.quantize_mxfp4(x.resolve_neg())
    for call in (lambda: cb.quantize_mxfp4(x), lambda: cb.linear_mxfp4(x, q, s), lambda: cb.linear_mxfp4(x.resolve_neg(), q, s, x[0]),
                 lambda: cb.gemm_mxfp4(q, s, q, s, torch.float32, out=x)):
        with pytest.raises(ValueError):
            call()
    assert same(cb.dequantize_mxfp4(q, s, 64, torch.float32), -torch.ones((64, 64), device=device))


def test_results_do_not_share_memory_with_operands(cb, device):
    x = torch.zeros((256, 256), device=device)
    q, s = cb.quantize_mxfp4(x)  # q [256, 128] bytes
    bias = torch.zeros(256 * 256, device=device)
    room = torch.zeros(2 * 256 * 256, device=device)
    for call in (lambda: cb.linear_mxfp4(x, q, s, out=x), lambda: cb.linear_mxfp4(x[:1], q, s, out=x[:1]),
                 lambda: cb.linear_mxfp4(x, q, s, bias[:256], out=bias.view(256, 256)),
                 lambda: cb.linear_mxfp4(room[:256 * 256].view(256, 256), q, s, out=room[256 * 255:256 * 511].view(256, 256)),
                 lambda: cb.gemm_mxfp4(q[:32], s[:1], q[:32], s[:1], torch.float16, out=q.view(torch.float16)[:16].view(32, 32)),
                 lambda: cb.dequantize_mxfp4(q[:1], s[:1], 256, torch.float16, out=q.view(torch.float16)[:4].view(1, 256))):
        with pytest.raises(ValueError, match="share memory"):
            call()
    y = cb.linear_mxfp4(room[:256 * 256].view(256, 256), q, s, out=room[256 * 256:].view(256, 256))  # neighbours
    assert y.data_ptr() == room.data_ptr() + 4 * 256 * 256 and not y.any()


# ------------------------------------------------------------------ what the documentation allows besides


def test_results_go_into_given_tensors(cb, device):
    (a, sa), (b, sb), want = exact_case(device, 70, 264, 320)
    out = torch.full((70, 264), float("nan"), device=device)
    assert cb.gemm_mxfp4(a, sa, b, sb, torch.float32, out=out) is not None and same(out, want)
    x, (w, sw), bias, sums = layer_case(device, torch.float16, 9, 320, 72)
    y = torch.empty((9, 72), device=device, dtype=torch.float16)
    cb.linear_mxfp4(x, w, sw, bias=bias, relu=False, out=y)
    assert same(y, (sums + bias.double()).half())
    q, s = cb.quantize_mxfp4(x=x, along=0)
    back = torch.empty((9, 320), device=device, dtype=torch.bfloat16)
    cb.dequantize_mxfp4(q, s, K=320, dtype=torch.bfloat16, out=back)
    assert same(back, plain.values(*plain.unpack(q, s)).bfloat16())


@pytest.mark.parametrize("n", [5, 130, 700])
def test_one_matrix_as_both_operands(cb, device, n):
    """A product of a matrix with itself: the same tensors twice, and a symmetric result to the last bit."""
    g = generator(device, n)
    code, byte = plain.random_packed(n, 160, -1, 1, g)
    q, s = plain.pack(code, byte)
    got = cb.gemm_mxfp4(q, s, q, s, torch.float32)
    v = plain.values(code, byte)
    assert same(got, v @ v.t()) and torch.equal(got, got.t())
    cb.check_device()


def test_garbage_behind_the_matrix_does_not_matter(cb, device):
    """Packed rows in the middle of a larger buffer whose other bytes are NaN scales and all codes."""
    from cudaintro_b200 import capi

    for M, N, K in ((3, 130, 96), (150, 40, 160), (300, 300, 256)):
        (a, sa), (b, sb), want = exact_case(device, M, N, K)
        held = []
        for t in (a, sa, b, sb):
            room = torch.full((t.numel() + 8192,), 255, dtype=torch.uint8, device=device)
            room[4096 : 4096 + t.numel()] = t.flatten()
            held.append(room)
        c = torch.empty((M, N), device=device)
        p = [r.data_ptr() + 4096 for r in held]
        assert capi.lib.b200_gemm_mxfp4(capi.F32, *p, c.data_ptr(), M, N, K, 0, torch.cuda.current_stream().cuda_stream) == 0
        cb.check_device()
        assert same(c, want)


def test_workspace_of_any_allowed_alignment(cb, device):
    from cudaintro_b200 import capi

    x, (w, sw), bias, sums = layer_case(device, torch.bfloat16, 150, 800, 264)
    need = capi.lib.b200_linear_mxfp4_workspace(150, 800, 264)
    assert need > 0
    for shift in (0, 16, 48, 240):
        room = torch.full((need + 512,), 255, dtype=torch.uint8, device=device)
        y = torch.empty((150, 264), dtype=torch.bfloat16, device=device)
        assert room.data_ptr() % 512 == 0
        rc = capi.lib.b200_linear_mxfp4(capi.BF16, x.data_ptr(), w.data_ptr(), sw.data_ptr(), bias.data_ptr(), y.data_ptr(), 150, 800,
                                        264, 0, room.data_ptr() + shift, need, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        cb.check_device()
        assert same(y, (sums + bias.double()).bfloat16())
        assert (room[:shift] == 255).all() and (room[shift + need :] == 255).all()


def test_layers_longer_than_a_launch_quantises(cb, device):
    """Rows too long, or too many, for the product to quantise them itself, at the borders of that rule."""
    for batch, in_f in ((16, 4096), (17, 4096), (17, 7712), (32, 4096), (33, 1024), (64, 1024), (1, 65536), (1, 65568), (2, 70000)):
        g = generator(device, batch + in_f)
        code, byte = plain.random_packed(batch, in_f, 0, 0, g)
        code[:, 0::32] = 7
        x = plain.values(code, byte)[:, :in_f].float()
        w = plain.random_packed(24, in_f, 0, 0, g)
        w[0][:, 4096:] = 0  # few terms, so that fp32 holds the sums
        y = cb.linear_mxfp4(x, *plain.pack(*w))
        cb.check_device()
        assert same(y, x.double() @ plain.values(*w)[:, :in_f].t())


@pytest.mark.parametrize("shape", [(300, 520, 768), (2304, 2304, 768), (40, 300, 768), (8, 264, 4096), (900, 16, 4096), (200, 300, 4096)])
def test_a_lost_arrival_is_reported_and_the_next_call_is_right(cb, device, shape):
    """Every wait is bounded: with one k-block's loads left out in the first CTA the product gives up after the 50 ms it is
    given here, says so, and works again.  CTA pairs, single CTAs, and clusters that split K."""
    import time

    from cudaintro_b200 import capi

    M, N, K = shape
    (a, sa), (b, sb), want = exact_case(device, M, N, K)
    assert same(cb.gemm_mxfp4(a, sa, b, sb, torch.float32), want)
    cb.check_device()
    try:
        capi._check(capi.lib.b200_test_lose_arrival(1, 50_000_000))
        t0 = time.perf_counter()
        cb.gemm_mxfp4(a, sa, b, sb, torch.float32)
        with pytest.raises(cb.B200Error) as info:
            cb.check_device()
        assert info.value.status == 4 and 0.04 <= time.perf_counter() - t0 < 2.0
    finally:
        capi._check(capi.lib.b200_test_lose_arrival(-1, 0))
    cb.check_device()
    for _ in range(2):
        assert same(cb.gemm_mxfp4(a, sa, b, sb, torch.float32), want)
    cb.check_device()


def test_offsets_beyond_32_bits(cb, device):
    """A matrix of 4.7e9 elements there and back, and a product with 4.4e9 results: first, middle and last rows."""
    if torch.cuda.mem_get_info(device)[0] < 60e9:
        pytest.skip("needs 60 GB of free device memory")
    rows, K = 36000, 131072
    g = generator(device, 2)
    x = torch.empty((rows, K), dtype=torch.bfloat16, device=device)
    picks = [0, 1, 16385, 32768, 35999]
    x.normal_(generator=g)
    q, s = cb.quantize_mxfp4(x)
    back = cb.dequantize_mxfp4(q, s, K, torch.bfloat16)
    want = plain.values(*plain.quantize(x[picks])).bfloat16()
    assert same(back[picks], want)
    del back, q, s
    # the same memory as columns: K = 36000 down, the last columns' elements lie beyond 2^32
    q, s = cb.quantize_mxfp4(x, 1)
    assert tuple(q.shape) == (K, 18000)
    cols = [0, 65536, K - 1]
    code, byte = plain.quantize(x[:, cols].t())
    got = torch.stack([torch.stack([q[c] & 15, q[c] >> 4], -1).flatten() for c in cols])
    assert torch.equal(got.long(), code)
    del x, q, s
    n = 66000
    a, sa = plain.pack(*plain.random_packed(n, 64, -1, 1, g))
    c = cb.gemm_mxfp4(a, sa, a, sa)
    cb.check_device()
    v = plain.values(*plain.unpack(a, sa))
    for r in (0, 32769, 65074, n - 1):
        assert same(c[r], (v @ v[r]).bfloat16())


def test_plain_launches_give_the_same(cb, device):
    """Without programmatic stream serialisation."""
    from cudaintro_b200 import capi

    def everything():
        out = []
        for shape in ((8, 264, 2048), (300, 520, 4096), (2304, 2304, 256)):
            (a, sa), (b, sb), want = exact_case(device, *shape)
            got = cb.gemm_mxfp4(a, sa, b, sb, torch.float32)
            assert same(got, want)
            out += [got, *cb.quantize_mxfp4(got), cb.linear_mxfp4(got, *cb.quantize_mxfp4(got))]
        return out

    first = everything()
    try:
        capi.lib.b200_set_dependent_launch(0)
        second = everything()
    finally:
        capi.lib.b200_set_dependent_launch(1)
    cb.check_device()
    assert all(torch.equal(x, y) for x, y in zip(first, second))


def test_host_threads_at_once(cb, device):
    """Four host threads, a stream and a shape each, the same thread-local and shared state underneath."""
    import threading

    shapes = [(1, 2048, 1024), (20, 1024, 520), (130, 2048, 264), (300, 4096, 520)]
    cases = [layer_case(device, torch.bfloat16, *s) for s in shapes]
    torch.cuda.synchronize()
    wrong = []

    def work(x, w, bias, sums):
        want = (sums + bias.double()).bfloat16()
        with torch.cuda.stream(torch.cuda.Stream()):
            ys = [cb.linear_mxfp4(x, *w, bias) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
            wrong.extend(i for i, y in enumerate(ys) if not same(y, want))

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    cb.check_device()
    assert not wrong
