"""CPU tests of the MXFP4 entry points: sizes, and refusals that come before any CUDA call."""
import ctypes as C

import pytest

import mxfp4_plain as plain

torch = pytest.importorskip("torch")


def test_sizes_of_packed_arrays(cb):
    from cudaintro_b200 import capi

    lib = capi.lib
    assert [lib.b200_mxfp4_row_bytes(k) for k in (0, 1, 32, 33, 784, 8192)] == [0, 16, 16, 32, 400, 4096]
    assert lib.b200_mxfp4_scale_bytes(1, 1) == 512 and lib.b200_mxfp4_scale_bytes(128, 128) == 512
    assert lib.b200_mxfp4_scale_bytes(129, 128) == 1024 and lib.b200_mxfp4_scale_bytes(129, 129) == 2048
    assert lib.b200_mxfp4_scale_bytes(0, 5) == 0 and lib.b200_mxfp4_scale_bytes(5, -1) == 0
    assert lib.b200_mxfp4_scale_bytes(1 << 30, 1 << 30) == 1 << 55  # no 32-bit wrap
    assert lib.b200_linear_mxfp4_workspace(200, 784, 10) >= 200 * 400 + 14 * 512
    assert lib.b200_linear_mxfp4_workspace(1, 4096, 11008) == 0 and lib.b200_linear_mxfp4_workspace(1, 1 << 20, 10) > 0
    assert lib.b200_linear_mxfp4_workspace(1, 4096, 28672) > 0
    assert lib.b200_linear_mxfp4_workspace(0, 784, 10) == 0


def test_plain_form_packs_and_unpacks():
    """The tests' own reference: packing is undone by unpacking, and known values round as the format says."""
    g = torch.Generator().manual_seed(1)
    code, byte = plain.random_packed(131, 200, -5, 5, g)
    got = plain.unpack(*plain.pack(code, byte))
    assert torch.equal(got[0], code) and torch.equal(got[1], byte)
    x = torch.zeros(1, 32)
    x[0, :12] = torch.tensor([7.0, 6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.2, -5.5, 4.5])
    code, byte = plain.quantize(x)
    assert byte.tolist() == [[127]]
    assert plain.values(code, byte)[0, :12].tolist() == [6, 6, 4, 4, 2, 2, 1, 1, 0, 0, -6, 4]


def test_refusals(cb):
    from cudaintro_b200 import capi

    lib, one, odd = capi.lib, C.c_void_p(64), C.c_void_p(65)
    f32, bf16, i8 = capi.F32, capi.BF16, capi.I8

    def quant(dtype=f32, x=one, q=one, s=one, R=4, Cc=64, ldx=0, along=0):
        return lib.b200_quantize_mxfp4(dtype, x, q, s, R, Cc, ldx, along, None)

    def dequant(dtype=f32, q=one, s=one, x=one, rows=4, K=64, ldx=0):
        return lib.b200_dequantize_mxfp4(dtype, q, s, x, rows, K, ldx, None)

    def gemm(dtype=bf16, a=one, sa=one, b=one, sb=one, c=one, M=4, N=4, K=64, ldc=0):
        return lib.b200_gemm_mxfp4(dtype, a, sa, b, sb, c, M, N, K, ldc, None)

    def linear(dtype=bf16, x=one, w=one, sw=one, bias=None, y=one, batch=200, i=64, o=4, flags=0, ws=one, n=1 << 20):
        return lib.b200_linear_mxfp4(dtype, x, w, sw, bias, y, batch, i, o, flags, ws, n, None)

    big = (1 << 30) + 1
    for call, wrong in (
        (quant, [dict(dtype=i8), dict(dtype=9), dict(x=None), dict(q=None), dict(s=None), dict(R=0), dict(Cc=-1), dict(ldx=63),
                 dict(along=2), dict(along=-1)]),
        (dequant, [dict(dtype=i8), dict(x=None), dict(q=None), dict(s=None), dict(rows=0), dict(K=0), dict(ldx=63)]),
        (gemm, [dict(dtype=i8), dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(c=None), dict(M=0), dict(N=0),
                dict(K=0), dict(ldc=3)]),
        (linear, [dict(dtype=i8), dict(x=None), dict(w=None), dict(sw=None), dict(y=None), dict(batch=0), dict(i=0), dict(o=0),
                  dict(flags=4), dict(ws=None), dict(n=0), dict(n=lib.b200_linear_mxfp4_workspace(200, 64, 4) - 1), dict(ws=odd)]),
    ):
        for kw in wrong:
            assert call(**kw) == 1, (call.__name__, kw)
            assert lib.b200_last_error()
    for call, wrong in (
        (quant, [dict(q=odd), dict(s=C.c_void_p(72)), dict(x=odd), dict(dtype=bf16, x=odd)]),
        (dequant, [dict(q=odd), dict(s=odd), dict(x=odd)]),
        (gemm, [dict(a=odd), dict(sa=odd), dict(b=odd), dict(sb=odd), dict(c=odd)]),
        (linear, [dict(w=odd), dict(sw=odd), dict(x=odd), dict(y=odd), dict(bias=odd)]),
    ):
        for kw in wrong:
            assert call(**kw) == 2, (call.__name__, kw)
    assert quant(R=big) == 5 and dequant(K=big, ldx=big) == 5 and gemm(M=big) == 5 and gemm(K=big) == 5 and linear(o=big) == 5


def test_rows_that_are_too_long_are_refused_with_their_limit(cb):
    from cudaintro_b200 import capi

    lib, one, longest = capi.lib, C.c_void_p(64), (1 << 28) - 4096
    assert lib.b200_quantize_mxfp4(capi.F32, one, one, one, 1, longest + 1, 0, 0, None) == 5
    assert str(longest).encode() in lib.b200_last_error()
    assert lib.b200_dequantize_mxfp4(capi.F32, one, one, one, 1, longest + 1, 0, None) == 5
    assert str(longest).encode() in lib.b200_last_error()


def test_no_cpu_fallback(cb):
    if torch.cuda.is_available():
        pytest.skip("this check is for machines without a GPU")
    with pytest.raises(ValueError):
        cb.quantize_mxfp4(torch.zeros(4, 64))
    from cudaintro_b200 import capi

    one = C.c_void_p(64)
    assert capi.lib.b200_gemm_mxfp4(capi.BF16, one, one, one, one, one, 4, 4, 64, 0, None) == 3
    assert capi.lib.b200_quantize_mxfp4(capi.F32, one, one, one, 4, 64, 0, 0, None) == 3
