"""MXFP4 quantiser, product and their values against plain 64-bit forms."""
import operator_refs as R
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def acts(m, k, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=g)
    x[:, ::37] *= 20.0
    return x.to(torch.bfloat16)


def families(m, k):
    """Values where the format can go wrong: ties of every step, block maxima at and next to powers
    of two, zeros, subnormals, the largest and smallest magnitudes."""
    g = torch.Generator().manual_seed(m * 7 + k)
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.96875, 4.0, -0.25, -0.75, -1.25, -5.0])
    ties = steps[torch.randint(0, len(steps), (m, k), generator=g)] * torch.exp2(torch.randint(-30, 30, (m, k // 32), generator=g).float()).repeat_interleave(32, 1)
    powers = torch.exp2(torch.randint(-126, 127, (m, k), generator=g).float()) * torch.where(torch.rand((m, k), generator=g) < 0.5, -1.0, 1.0)
    tiny = torch.randint(-200, 201, (m, k), generator=g).float() * 2.0 ** -133
    sparse = torch.where(torch.rand((m, k), generator=g) < 0.03, torch.randn((m, k), generator=g), 0.0)
    return {"normal": acts(m, k, k), "ties": ties.to(torch.bfloat16), "powers": powers.to(torch.bfloat16), "tiny": tiny.to(torch.bfloat16),
            "sparse": sparse.to(torch.bfloat16), "zeros": torch.zeros((m, k), dtype=torch.bfloat16),
            "largest": (torch.sign(torch.randn((m, k), generator=g)) * torch.finfo(torch.bfloat16).max).to(torch.bfloat16)}


@pytest.mark.parametrize("m,k", [(1, 32), (3, 64), (127, 160), (128, 128), (129, 2080), (300, 416)])
def test_quantizer_is_exact(cuda_pkg, m, k):
    for name, x in families(m, k).items():
        code, byte = R.mx_quantize(x.double())
        q, s = cuda_pkg.ops.quantize_mxfp4(x.to(DEV))
        q, s = q.cpu(), s.cpu()
        assert q.shape == (m, k // 2) and tuple(s.shape) == cuda_pkg.ops.mxfp4_scale_shape(m, k)
        assert torch.equal(s, R.mx_tiles(byte)), name            # the bytes outside the matrix too
        assert torch.equal(R.mx_codes(q), code), name
        back = cuda_pkg.ops.dequantize_mxfp4(q.to(DEV), s.to(DEV)).cpu()
        assert torch.equal(back.double(), R.mx_values(code, byte)), name   # exact in bf16


def test_quantizer_blocks_with_nan_or_infinity(cuda_pkg):
    x = acts(5, 160, 1)
    x[1, 40], x[2, 0], x[3, 159] = float("nan"), float("inf"), float("-inf")
    bad = {(1, 1), (2, 0), (3, 4)}
    q, s = cuda_pkg.ops.quantize_mxfp4(x.to(DEV))
    byte, code = R.mx_bytes(s.cpu(), 5, 160), R.mx_codes(q.cpu())
    want_code, want_byte = R.mx_quantize(torch.nan_to_num(x.double(), 0.0, 0.0, 0.0))
    values = cuda_pkg.ops.dequantize_mxfp4(q, s).cpu().float()
    for r in range(5):
        for b in range(5):
            part = slice(32 * b, 32 * b + 32)
            if (r, b) in bad:
                assert byte[r, b] == 255 and (code[r, part] == 0).all() and torch.isnan(values[r, part]).all()
            else:
                assert byte[r, b] == want_byte[r, b] and torch.equal(code[r, part], want_code[r, part])


def near_border(y, byte, code, delta):
    """Every code is the rounding of y moved by at most `delta` of itself, every byte that of a
    largest magnitude moved as much."""
    blocks = y.view(y.shape[0], -1, 32)
    big = blocks.abs().amax(-1)
    low, high = R.mx_byte(big * (1 - delta)), R.mx_byte(big * (1 + delta))
    assert ((byte == low) | (byte == high)).all()
    unit = torch.exp2((byte - 127).double())[..., None]
    c = code.view(blocks.shape)
    a, b = R.mx_elements(blocks * (1 - delta), unit), R.mx_elements(blocks * (1 + delta), unit)
    assert (((c & 7) == a) | ((c & 7) == b)).all()
    signed = (c & 7) > 0
    assert torch.equal(c[signed] >= 8, torch.signbit(blocks)[signed])


@pytest.mark.parametrize("m,k", [(1, 32), (130, 96), (257, 1024)])
def test_swiglu_quantizer(cuda_pkg, m, k):
    x = acts(m, 2 * k, m + k)
    x[:, :k].clamp_(-60, 60)
    g, u = x[:, :k].double(), x[:, k:].double()
    q, s = cuda_pkg.ops.swiglu_quantize_mxfp4(x.to(DEV))
    # the fast exponential is within 2 + 1.173 |g| units of 2^-23 (|g| <= 60: 73), the reciprocal,
    # the sum and the two products within one each: 78 * 2^-23 < 1e-5
    near_border(g * torch.sigmoid(g) * u, R.mx_bytes(s.cpu(), m, k), R.mx_codes(q.cpu()), 1e-5)


@pytest.mark.parametrize("m,k", [(1, 8), (5, 3), (77, 1000), (33, 2080), (300, 4096), (1, 1), (100, 7), (65, 1001), (9, 4099)])
def test_int8_values(cuda_pkg, m, k):
    g = torch.Generator().manual_seed(m + k)
    q = torch.randint(-128, 128, (m, k), dtype=torch.int8, generator=g)
    s = torch.rand((m, 1), generator=g) * 0.1
    got = cuda_pkg.ops.dequantize_int8_rowwise(q.to(DEV), s.to(DEV)).cpu()
    assert torch.equal(got, (q.float() * s).to(torch.bfloat16))


def product_bound(a, w, want):
    """One rounding to bf16, and fp32 sums: every 32 products may lose one unit of 2^-23 of the
    largest partial sum, which the sum of magnitudes bounds."""
    return R.BF16_HALF * want.abs() + (a.shape[1] / 32 + 2) * 2.0 ** -23 * (a.abs() @ w.abs().T) + 1e-38


@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (1, 264, 4096), (3, 16, 64), (16, 520, 96), (31, 1000, 256), (64, 256, 544),
                                   (65, 128, 512), (128, 256, 256), (129, 264, 288), (200, 384, 2080), (256, 512, 1024),
                                   (257, 648, 416), (1000, 1000, 1056), (2049, 2312, 4128), (65, 19464, 96)])
@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float32])
def test_product(cuda_pkg, m, n, k, bias):
    a, sa, av = (t.to(DEV) for t in R.random_mx(m, k, m + k))
    w, sw, wv = (t.to(DEV) for t in R.random_mx(n, k, n + k + 1))
    b = None if bias is None else (torch.randn(n, generator=torch.Generator().manual_seed(n)) * 10).to(bias).to(DEV)
    got = cuda_pkg.ops.mxfp4_gemm(a, sa, w, sw, b)
    again = cuda_pkg.ops.mxfp4_gemm(a, sa, w, sw, b)
    cuda_pkg.ops.check_device_status()
    want = av @ wv.T if b is None else av @ wv.T + b.double()
    bound = product_bound(av, wv, want)
    if b is not None:
        bound = bound + 2.0 ** -23 * b.double().abs()
    over = ((got.double() - want).abs() > bound).sum()
    assert got.shape == (m, n) and int(over) == 0, (int(over), float(((got.double() - want).abs() / bound).max()))
    assert torch.equal(got, again)                              # deterministic


def test_product_every_scale_and_nan(cuda_pkg):
    """Scales over the whole range that bf16 can answer, and blocks with the NaN byte."""
    a, sa, av = (t.to(DEV) for t in R.random_mx(140, 320, 5, 64, 190))
    w, sw, wv = (t.to(DEV) for t in R.random_mx(72, 320, 6, 100, 154))
    got = cuda_pkg.ops.mxfp4_gemm(a, sa, w, sw).double()
    want = av @ wv.T
    assert ((got - want).abs() <= product_bound(av, wv, want)).all()
    byte = R.mx_bytes(sa.cpu(), 140, 320)
    byte[3, 2] = byte[139, 9] = 255
    got = cuda_pkg.ops.mxfp4_gemm(a, R.mx_tiles(byte).to(DEV), w, sw).double()
    rows = torch.isnan(got).all(1).nonzero()[:, 0].tolist()
    assert rows == [3, 139]
    keep = [r for r in range(140) if r not in rows]
    assert ((got - want).abs() <= product_bound(av, wv, want))[keep].all()


@pytest.mark.parametrize("act", [None, "swiglu"])
@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (7, 264, 128), (300, 264, 512)])
def test_linear_is_quantizer_and_product(cuda_pkg, m, n, k, act):
    ops = cuda_pkg.ops
    x = acts(m, 2 * k if act else k, m).to(DEV)
    w, sw, _ = R.random_mx(n, k, n)
    w, sw = w.to(DEV), sw.to(DEV)
    b = torch.randn(n, device=DEV).to(torch.bfloat16)
    q, s = (ops.swiglu_quantize_mxfp4 if act else ops.quantize_mxfp4)(x)
    assert torch.equal(ops.mxfp4_linear(x, w, sw, b, input_act=act), ops.mxfp4_gemm(q, s, w, sw, b))


def test_empty_sizes(cuda_pkg):
    ops = cuda_pkg.ops
    e = lambda *s: torch.empty(s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    q, s = ops.quantize_mxfp4(e(0, 64))
    assert q.shape == (0, 32) and s.shape == (0, 1, 512) and ops.dequantize_mxfp4(q, s).shape == (0, 64)
    w, sw, _ = R.random_mx(8, 64, 1)
    assert ops.mxfp4_gemm(q, s, w.to(DEV), sw.to(DEV)).shape == (0, 8)
    assert ops.mxfp4_linear(e(0, 64), w.to(DEV), sw.to(DEV)).shape == (0, 8)
    assert ops.dequantize_int8_rowwise(torch.empty((0, 5), dtype=torch.int8, device=DEV), torch.empty(0, device=DEV)).shape == (0, 5)


def test_refusals(cuda_pkg):
    ops = cuda_pkg.ops
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=DEV)
    q, s = ops.quantize_mxfp4(x)
    w, sw = (t.to(DEV) for t in R.random_mx(8, 64, 1)[:2])
    for call, match in [(lambda: ops.quantize_mxfp4(x[:, :48].contiguous()), "multiple of 32"),
                        (lambda: ops.quantize_mxfp4(x[:, ::2]), "contiguous"),
                        (lambda: ops.quantize_mxfp4(x.float()), "bfloat16"),
                        (lambda: ops.swiglu_quantize_mxfp4(x[:, :32].contiguous()), "multiple of 64"),
                        (lambda: ops.dequantize_mxfp4(q, s[:, :, :256].contiguous()), "scales of the matrix"),
                        (lambda: ops.mxfp4_gemm(q, s, w[:, :16].contiguous(), sw), "shape mismatch"),
                        (lambda: ops.mxfp4_gemm(q, s, w[:4].contiguous(), sw), "multiple of 8"),
                        (lambda: ops.mxfp4_gemm(q, s, w, sw, torch.zeros(7, device=DEV)), "exactly N values"),
                        (lambda: ops.mxfp4_gemm(q, s, w, sw, torch.zeros(8, dtype=torch.float16, device=DEV)), "float32"),
                        (lambda: ops.mxfp4_linear(x, w, sw, input_act="gelu"), "unknown input activation")]:
        with pytest.raises(RuntimeError, match=match):
            call()
    with pytest.raises(ValueError, match="inner dimensions"):
        ops.mxfp4_linear(x[:, :32].contiguous(), w, sw)


def test_side_stream_and_captured_graph(cuda_pkg):
    """The linear on a stream of its own, and captured once and replayed on other inputs."""
    ops = cuda_pkg.ops
    w, sw = (t.to(DEV) for t in R.random_mx(264, 512, 1)[:2])
    b = torch.randn(264, device=DEV)
    xs = [acts(m, 512, m).to(DEV) for m in (300, 300, 300)]
    want = [ops.mxfp4_linear(x, w, sw, b) for x in xs]
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.mxfp4_linear(x, w, sw, b) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, t) for g, t in zip(got, want))
    static = xs[0].clone()
    graphs = []
    for _ in range(2):                                          # two captures of the same call
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.mxfp4_linear(static, w, sw, b)
        graphs.append((graph, out))
    for x, t in zip(xs, want):
        static.copy_(x)
        for graph, _ in graphs:
            graph.replay()
        assert all(torch.equal(out, t) for _, out in graphs)


def test_offsets_past_32_bits(cuda_pkg):
    """More than 2^31 elements: the last rows are quantised like the same rows alone."""
    ops = cuda_pkg.ops
    m, k = 263000, 8192
    x = torch.zeros((m, k), dtype=torch.bfloat16, device=DEV)
    x[-300:] = torch.randn((300, k), device=DEV).to(torch.bfloat16)
    first = (m - 300) // 128 * 128                              # whole scale tiles
    q, s = ops.quantize_mxfp4(x)
    q2, s2 = ops.quantize_mxfp4(x[first:].contiguous())
    assert torch.equal(q[first:], q2) and torch.equal(s[first // 128:], s2)
    back = ops.dequantize_mxfp4(q, s)
    assert torch.equal(back[first:], ops.dequantize_mxfp4(q2, s2)) and not back[:first].any()


def test_swiglu_columns_behind_the_gates_are_not_read_as_gates(cuda_pkg):
    """K not a multiple of 128: the columns behind the last gate are up columns; infinities there
    stay in their own blocks and the scale bytes outside the matrix are 0."""
    m, k = 140, 160
    x = acts(m, 2 * k, 3).clamp(-20, 20)
    want_q, want_s = (t.cpu() for t in cuda_pkg.ops.swiglu_quantize_mxfp4(x.to(DEV)))
    x[5, k + 3] = float("inf")
    q, s = (t.cpu() for t in cuda_pkg.ops.swiglu_quantize_mxfp4(x.to(DEV)))
    byte, want = R.mx_bytes(s, m, k), R.mx_bytes(want_s, m, k)
    assert byte[5, 0] == 255
    byte[5, 0] = want[5, 0]
    assert torch.equal(byte, want) and torch.equal(R.mx_tiles(byte), want_s)
    assert torch.equal(q[:, 16:], want_q[:, 16:]) and not q[5, :16].any()
