"""The transformer-block operators without a GPU: the C ABI refuses bad arguments before any launch,
the Python entry points refuse CPU tensors, and the plain forms that the GPU tests compare with
agree with the format's definition."""
import ctypes

import operator_refs as R
import pytest
import torch

P = ctypes.c_void_p
FAKE, OTHER, ODD = P(0x1000), P(0x2000), P(0x1001)   # never dereferenced


def test_mxfp4_arguments_are_checked_before_launch(pkg):
    lib = pkg._lib.load()
    for name in ("b2_quantize_mxfp4", "b2_swiglu_quantize_mxfp4", "b2_dequantize_mxfp4"):
        f = getattr(lib, name)
        assert f(FAKE, FAKE, FAKE, -1, 64, None) == 2
        assert f(FAKE, FAKE, FAKE, 4, 48, None) == 4
        assert b"multiple of 32" in lib.b2_last_error()
        assert f(FAKE, None, FAKE, 4, 64, None) == 7
        assert f(FAKE, FAKE, ODD, 4, 64, None) == 3
        assert f(ODD, FAKE, FAKE, 4, 64, None) == 3
        assert f(FAKE, FAKE, FAKE, 0, 64, None) == 0 and f(FAKE, FAKE, FAKE, 4, 0, None) == 0
        assert f(FAKE, FAKE, FAKE, 1 << 40, 64, None) == 8
    assert lib.b2_dequantize_int8_rowwise(FAKE, None, FAKE, 4, 4, None) == 7
    assert lib.b2_dequantize_int8_rowwise(FAKE, ODD, FAKE, 4, 4, None) == 3
    assert lib.b2_dequantize_int8_rowwise(FAKE, FAKE, FAKE, 0, 4, None) == 0
    g = lib.b2_mxfp4_gemm
    assert g(FAKE, FAKE, FAKE, FAKE, None, 3, FAKE, 8, 8, 64, None) == 1
    assert g(FAKE, FAKE, FAKE, FAKE, None, 0, FAKE, 8, 8, 48, None) == 4
    assert g(FAKE, FAKE, FAKE, FAKE, None, 0, FAKE, 8, 12, 64, None) == 4
    assert g(FAKE, FAKE, FAKE, FAKE, None, 0, FAKE, 8, 8, 0, None) == 2
    assert g(FAKE, FAKE, FAKE, FAKE, None, 0, FAKE, -8, 8, 64, None) == 2
    assert g(FAKE, None, FAKE, FAKE, None, 0, FAKE, 8, 8, 64, None) == 7
    assert g(FAKE, FAKE, FAKE, FAKE, None, 1, FAKE, 8, 8, 64, None) == 7
    assert g(FAKE, FAKE, FAKE, ODD, None, 0, FAKE, 8, 8, 64, None) == 3
    assert g(FAKE, FAKE, FAKE, FAKE, ODD, 2, FAKE, 8, 8, 64, None) == 3
    assert g(FAKE, FAKE, FAKE, FAKE, None, 0, FAKE, 0, 8, 64, None) == 0
    assert g(FAKE, FAKE, FAKE, FAKE, None, 0, FAKE, 1 << 33, 8, 64, None) == 8
    l = lib.b2_mxfp4_linear
    assert l(FAKE, 5, FAKE, FAKE, None, 0, FAKE, FAKE, FAKE, 8, 8, 64, None) == 1
    assert l(None, 0, FAKE, FAKE, None, 0, FAKE, FAKE, FAKE, 8, 8, 64, None) == 7
    assert l(FAKE, 0, FAKE, FAKE, None, 0, FAKE, None, FAKE, 8, 8, 64, None) == 7
    assert l(FAKE, 0, FAKE, FAKE, None, 0, FAKE, FAKE, FAKE, 8, 0, 64, None) == 0


def test_rmsnorm_arguments_are_checked_before_launch(pkg):
    lib = pkg._lib.load()
    for f in (lib.b2_rmsnorm_residual_quant, lib.b2_rmsnorm_residual_mxfp4):
        assert f(FAKE, FAKE, FAKE, OTHER, FAKE, FAKE, 4, 0, 1e-6, None) == 2
        assert f(FAKE, FAKE, FAKE, OTHER, FAKE, FAKE, 4, 64, float("nan"), None) == 2
        assert f(FAKE, FAKE, FAKE, OTHER, FAKE, FAKE, 4, 64, float("inf"), None) == 2
        assert f(FAKE, None, FAKE, OTHER, FAKE, FAKE, 4, 64, 1e-6, None) == 7    # a sum without a residual
        assert f(FAKE, FAKE, FAKE, None, FAKE, FAKE, 4, 64, 1e-6, None) == 7
        assert f(FAKE, OTHER, FAKE, FAKE, FAKE, FAKE, 4, 64, 1e-6, None) == 3    # sum aliases x
        assert f(FAKE, OTHER, FAKE, OTHER, FAKE, FAKE, 4, 64, 1e-6, None) == 3   # sum aliases the residual
        assert f(ODD, None, FAKE, None, FAKE, FAKE, 4, 64, 1e-6, None) == 3
        assert f(FAKE, None, FAKE, None, FAKE, FAKE, 0, 64, 1e-6, None) == 0
    assert lib.b2_rmsnorm_residual_mxfp4(FAKE, None, FAKE, None, FAKE, FAKE, 4, 40, 1e-6, None) == 4
    assert lib.b2_rmsnorm_residual_mxfp4(FAKE, None, FAKE, None, FAKE, FAKE, 4, 16416, 1e-6, None) == 8


def test_entry_points_refuse_cpu_tensors(pkg):
    ops = pkg.ops
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    q, s = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 1, 512), dtype=torch.uint8)
    for call in (lambda: ops.quantize_mxfp4(x), lambda: ops.swiglu_quantize_mxfp4(x), lambda: ops.dequantize_mxfp4(q, s),
                 lambda: ops.mxfp4_gemm(q, s, q, s), lambda: ops.mxfp4_linear(x, q, s),
                 lambda: ops.dequantize_int8_rowwise(q.to(torch.int8), torch.zeros(4)),
                 lambda: ops.rmsnorm_residual_quant(x, None, x[0]), lambda: ops.rmsnorm_residual_mxfp4(x, x, x[0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_plain_mxfp4_follows_the_definition():
    x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.26, -0.24] + [0.0] * 22], dtype=torch.float64)
    code, byte = R.mx_quantize(x)
    assert byte.tolist() == [[127]]
    assert R.mx_values(code, byte)[0, :10].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, -0.5, 0]
    for largest, want in [(1.0, 125), (1.999, 125), (2.0, 126), (0.0, 0), (2.0 ** -140, 0), (2.0 ** -125, 0), (2.0 ** -124, 1), (3e38, 252)]:
        assert int(R.mx_byte(torch.tensor(largest, dtype=torch.float64))) == want, largest
    byte = torch.randint(0, 255, (300, 9))
    assert torch.equal(R.mx_bytes(R.mx_tiles(byte), 300, 288), byte)
    codes = torch.randint(0, 16, (5, 64))
    assert torch.equal(R.mx_codes(R.mx_pack(codes)), codes)


def test_window_arguments_are_checked_before_launch(pkg):
    lib = pkg._lib.load()
    s = [1 << 20, 128, 128 * 4]
    good = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, ws=None, ws_bytes=0, lengths=None, B=1, H=4, Hkv=4, Sq=512, Sk=512, qs=s, ks=s,
                vs=s, scale=0.1, left=1, right=1, sinks=0)

    def call(**change):
        a = {**good, **change}
        return lib.b2_window_fwd(a["q"], a["k"], a["v"], a["out"], a["ws"], a["ws_bytes"], a["lengths"], a["B"], a["H"], a["Hkv"],
                                 a["Sq"], a["Sk"], *a["qs"], *a["ks"], *a["vs"], a["scale"], a["left"], a["right"], a["sinks"], None)

    assert call(B=0) == 2 and call(Sk=0) == 2 and call(Sq=-1) == 2 and call(Hkv=3) == 2
    assert b"no multiple" in lib.b2_last_error()
    assert call(left=-2) == 2 and call(right=-2) == 2 and call(sinks=-1) == 2
    assert call(scale=float("nan")) == 2 and call(scale=0.0) == 2
    assert call(k=None) == 7 and call(out=None) == 7
    assert call(v=ODD) == 3 and call(lengths=ODD) == 3
    assert call(ks=[1 << 20, 100, 512]) == 3 and call(vs=[1 << 20, 0, 512]) == 3 and call(qs=[1 << 20, -128, 512]) == 3
    assert call(ks=[1 << 20, 1 << 38, 512]) == 8 and call(B=65536) == 8 and call(Sq=1 << 29) == 8
    # single tokens of a few heads over a very long cache leave their parts in memory
    need = ctypes.c_int64(-1)
    assert lib.b2_window_fwd_workspace(1, 2, 2, 1, 65536, -1, 0, 0, ctypes.byref(need)) == 0 and need.value > 0
    assert call(H=2, Hkv=2, Sq=1, Sk=65536, left=-1, right=0, ws=FAKE, ws_bytes=need.value - 1) == 2
    assert b"workspace" in lib.b2_last_error()
    assert lib.b2_window_fwd_workspace(8, 24, 24, 4096, 4096, -1, 0, 0, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.b2_window_fwd_workspace(1, 4, 4, 1, 8192, -1, 0, 0, None) == 7
    assert lib.b2_window_fwd_workspace(1, 4, 3, 1, 8192, -1, 0, 0, ctypes.byref(need)) == 2
    x = torch.zeros((1, 2, 8, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.ops.window_fwd_bhsd(x, x, x, 0.1, -1, -1)
