"""RMSNorm with the residual's addition and a quantised output, against plain 64-bit forms."""
import operator_refs as R
import pytest
import torch
from test_gpu_mxfp4 import acts, near_border

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# y relative to the formula: the sum of squares has at most 64 terms added one after another in a
# thread (C <= 16384) and ten more levels, 74 * 2^-24, of which the square root halves; rsqrtf is
# within 2 units of 2^-23, the mean, eps and the two products within 2^-24 each: under 4e-6; the
# scale adds three roundings.
DELTA = 6e-6


def inputs(m, c, residual):
    x, r = acts(m, c, m + c), acts(m, c, m + c + 1) if residual else None
    w = (1 + 0.2 * torch.randn(c, generator=torch.Generator().manual_seed(c))).to(torch.bfloat16)
    return x, r, w


def dev(t):
    return None if t is None else t.to(DEV)


def check_int8(ops, x, r, w, eps):
    total, y = R.rmsnorm(x, r, w, eps)
    q, s, got = (t.cpu() for t in ops.rmsnorm_residual_quant(dev(x), dev(r), dev(w), eps))
    assert torch.equal(got, total)
    want = (y.abs().amax(1, keepdim=True) / 127).clamp(min=1e-30)
    assert ((s.double() - want).abs() <= DELTA * want).all()
    assert ((q.double() * s.double() - y).abs() <= s.double() * (0.5 + 127 * 2 * DELTA)).all()
    return q, s


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("m,c", [(1, 1), (1, 8), (3, 7), (2, 250), (300, 256), (9, 264), (130, 1024), (65, 1032), (33, 2048),
                                 (17, 2056), (70, 3072), (40, 4096), (21, 5120), (19, 8192), (11, 8200), (7, 16384),
                                 (5, 16392), (3, 20001), (200, 7),
                                 (129, 255), (64, 257), (33, 1001), (40, 1022), (17, 2047), (21, 2051), (9, 4095), (11, 8189),
                                 (5, 16375), (4, 16379)])
def test_int8(cuda_pkg, m, c, residual):
    check_int8(cuda_pkg.ops, *inputs(m, c, residual), 1e-6)


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("m,c", [(1, 32), (3, 96), (130, 256), (129, 1056), (257, 2080), (128, 3072), (40, 4096), (21, 5120),
                                 (19, 8192), (7, 16384)])
def test_mxfp4(cuda_pkg, m, c, residual):
    x, r, w = inputs(m, c, residual)
    total, y = R.rmsnorm(x, r, w, 1e-5)
    q, s, got = (t.cpu() for t in cuda_pkg.ops.rmsnorm_residual_mxfp4(dev(x), dev(r), dev(w), 1e-5))
    assert torch.equal(got, total)
    byte = R.mx_bytes(s, m, c)
    near_border(y, byte, R.mx_codes(q), DELTA)
    assert torch.equal(s, R.mx_tiles(byte))                     # zeros outside the matrix


@pytest.mark.parametrize("c", [264, 250])
def test_special_rows(cuda_pkg, c):
    """Zeros with and without eps, a lone huge or tiny value, NaN and infinities in x or residual."""
    ops = cuda_pkg.ops
    x, r, w = inputs(8, c, True)
    x[0], r[0] = 0, 0
    x[1], r[1] = 0, 0
    x[1, 5] = 1e18
    x[2], r[2] = 0, 0
    x[2, 7] = 1e-18
    check_int8(ops, x[:3].contiguous(), r[:3].contiguous(), w, 1e-6)
    x[4, 3], r[5, 2], x[6, 1] = float("nan"), float("inf"), float("-inf")
    x[7, 0], r[7, 0] = float("inf"), float("-inf")              # their sum is a NaN
    q, s, total = ops.rmsnorm_residual_quant(dev(x), dev(r), dev(w))
    q, s, total = q.cpu(), s.cpu(), total.cpu()
    assert torch.equal(total.isnan(), (x + r).isnan()) and torch.equal(total.isinf(), (x + r).isinf())
    assert torch.isfinite(s[:4]).all() and not torch.isfinite(s[4:]).any() and not q[4:].any()
    check_int8(ops, x[3:4].contiguous(), r[3:4].contiguous(), w, 1e-6)
    if c % 32 == 0:
        q, s, _ = ops.rmsnorm_residual_mxfp4(dev(x), dev(r), dev(w))
        byte = R.mx_bytes(s.cpu(), 8, c)
        assert (byte[:4] < 255).all() and (byte[4:] == 255).any(1).all()


def test_zero_rows_without_eps(cuda_pkg):
    """0 / sqrt(0) is a NaN in the formula; it stays one."""
    x, _, w = inputs(2, 64, False)
    x[1] = 0
    q, s, _ = cuda_pkg.ops.rmsnorm_residual_quant(dev(x), None, dev(w), 0.0)
    assert torch.isfinite(s[0]).all() and torch.isnan(s[1]).all() and not q[1].any()


def test_same_tensor_twice_and_inputs_kept(cuda_pkg):
    x, _, w = inputs(50, 512, False)
    xd = dev(x)
    q, s, total = cuda_pkg.ops.rmsnorm_residual_quant(xd, xd, dev(w))
    assert torch.equal(xd.cpu(), x) and torch.equal(total.cpu(), (x + x))
    q2, s2, total2 = cuda_pkg.ops.rmsnorm_residual_quant(xd, xd, dev(w))
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_many_rows(cuda_pkg):
    """More rows than the grid walks at once: every row as if alone."""
    ops = cuda_pkg.ops
    x, r, w = inputs(1, 256, True)
    m = 148 * 8 * 8 * 3 + 5
    g = torch.Generator().manual_seed(3)
    scale = torch.exp2(torch.randint(-3, 4, (m, 1), generator=g).float()).to(torch.bfloat16)
    q, s, _ = ops.rmsnorm_residual_quant(dev(x * scale), dev(r * scale), dev(w), 0.0)
    assert (q == q[0]).all()                                    # scaling by powers of two changes nothing without eps
    assert (s == s[0]).all()
    q, t, _ = ops.rmsnorm_residual_mxfp4(dev(x * scale), dev(r * scale), dev(w), 0.0)
    assert (q == q[0]).all()


@pytest.mark.parametrize("c", [1, 5, 63, 1001])
def test_odd_widths_stay_inside_the_tensors(cuda_pkg, c):
    """Rows that share vectors with their neighbours, in the middle of larger buffers that stay as
    they were; and tensors that start anywhere."""
    m = 37
    x, r, w = inputs(m, c, True)
    want = cuda_pkg.ops.rmsnorm_residual_quant(dev(x), dev(r), dev(w))
    for offset in (0, 8, 3):
        place = lambda t: torch.cat((torch.full((offset,), 7.0, dtype=t.dtype), t.flatten(), torch.full((9,), 7.0, dtype=t.dtype))).to(DEV)[offset:offset + t.numel()].view(t.shape)  # noqa: E731
        xo, ro, wo = place(x), place(r), place(w)
        q, s, total = cuda_pkg.ops.rmsnorm_residual_quant(xo, ro, wo)
        # another kernel may take over (pointers off a vector's start): the sums run in another order
        assert torch.equal(total, want[2])
        assert ((s - want[1]).abs() <= DELTA * want[1]).all() and ((q.int() - want[0].int()).abs() <= 1).all()
    lib = cuda_pkg._lib.load()
    stream = torch.cuda.current_stream(DEV).cuda_stream
    pad = 64
    total, q = (torch.full((m * c + 2 * pad,), 5, dtype=t, device=DEV) for t in (torch.bfloat16, torch.int8))
    scale = torch.zeros(m, device=DEV)
    xd, rd, wd = dev(x), dev(r), dev(w)
    assert lib.b2_rmsnorm_residual_quant(xd.data_ptr(), rd.data_ptr(), wd.data_ptr(), total.data_ptr() + 2 * pad, q.data_ptr() + pad,
                                         scale.data_ptr(), m, c, 1e-6, stream) == 0
    for t, inside in ((total, want[2]), (q, want[0])):
        assert (t[:pad] == 5).all() and (t[pad + m * c:] == 5).all() and torch.equal(t[pad:pad + m * c].view(m, c), inside)


def test_empty_and_refusals(cuda_pkg):
    ops = cuda_pkg.ops
    x, r, w = (dev(t) for t in inputs(4, 64, True))
    q, s, total = ops.rmsnorm_residual_quant(x[:0], r[:0], w)
    assert q.shape == (0, 64) and s.shape == (0, 1) and total.shape == (0, 64)
    assert ops.rmsnorm_residual_mxfp4(x[:0], None, w)[1].shape == (0, 1, 512)
    for call, match in [(lambda: ops.rmsnorm_residual_quant(x, r[:2], w), "residual"),
                        (lambda: ops.rmsnorm_residual_quant(x, r.float(), w), "residual"),
                        (lambda: ops.rmsnorm_residual_quant(x, r, w[:32]), "weight must contain"),
                        (lambda: ops.rmsnorm_residual_quant(x, r, w.float()), "weight must be bfloat16"),
                        (lambda: ops.rmsnorm_residual_quant(x.t(), None, w), "x must be"),
                        (lambda: ops.rmsnorm_residual_quant(x, r, w, float("nan")), "eps"),
                        (lambda: ops.rmsnorm_residual_quant(x, r, w, -1.0), "eps"),
                        (lambda: ops.rmsnorm_residual_mxfp4(x[:, :40].contiguous(), None, w[:40]), "multiple of 32"),
                        (lambda: ops.rmsnorm_residual_mxfp4(torch.zeros((2, 16416), dtype=torch.bfloat16, device=DEV), None,
                                                            torch.zeros(16416, dtype=torch.bfloat16, device=DEV)), "16384")]:
        with pytest.raises(RuntimeError, match=match):
            call()
