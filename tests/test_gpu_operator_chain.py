"""The transformer-block operators together, as a layer uses them: every stage against its plain
64-bit form on the inputs that the stage before produced, and the DiT block's options against the
calls that they stand for."""
import operator_refs as R
import pytest
import torch
from test_gpu_mxfp4 import near_border, product_bound
from test_gpu_rmsnorm import DELTA
from test_gpu_window import bound

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def weight(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((n, k), generator=g) * 0.05).to(torch.bfloat16).to(DEV)


def values(q, s):
    m, k = q.shape[0], q.shape[1] * 2
    return R.mx_values(R.mx_codes(q), R.mx_bytes(s, m, k))


def test_a_layer_over_a_cache(cuda_pkg):
    """Two sequences of different length take a chunk of five tokens through a layer: norm with the
    residual -> 4-bit projection -> keys and values into the cache -> windowed attention of shared
    heads -> 4-bit output projection -> norm with the residual -> int8 projection."""
    ops = cuda_pkg.ops
    B, T, C, H, Hkv, Sk = 2, 5, 512, 8, 2, 700
    g = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).to(DEV)  # noqa: E731
    x, res = rnd(B * T, C), rnd(B * T, C)
    w1, w2 = (1 + 0.1 * torch.randn(C, generator=g)).to(torch.bfloat16).to(DEV), (1 + 0.1 * torch.randn(C, generator=g)).to(torch.bfloat16).to(DEV)
    wqkv, wout = ops.quantize_mxfp4(weight((H + 2 * Hkv) * 128, C, 2)), ops.quantize_mxfp4(weight(C, H * 128, 3))
    k_cache, v_cache = rnd(B, Sk, Hkv, 128), rnd(B, Sk, Hkv, 128)
    lengths = torch.tensor([333, 700], dtype=torch.int32, device=DEV)    # with the chunk
    k_cache[0, 333:] = float("nan")                                      # not written yet
    v_cache[0, 333:] = float("nan")

    a, sa, total = ops.rmsnorm_residual_mxfp4(x, res, w1, 1e-6)
    want_total, y = R.rmsnorm(x, res, w1, 1e-6)
    assert torch.equal(total, want_total)
    near_border(y.cpu(), R.mx_bytes(sa.cpu(), B * T, C), R.mx_codes(a.cpu()), DELTA)

    qkv = ops.mxfp4_gemm(a, sa, *wqkv)
    av, wv = values(a, sa), values(*wqkv)
    assert ((qkv.double() - av @ wv.T).abs() <= product_bound(av, wv, av @ wv.T)).all()

    q, k, v = qkv.view(B, T, H + 2 * Hkv, 128).split((H, Hkv, Hkv), dim=2)
    for b, n in enumerate(lengths.tolist()):
        k_cache[b, n - T:n], v_cache[b, n - T:n] = k[b], v[b]
    heads = lambda t: t.transpose(1, 2)  # noqa: E731
    args = (heads(q), heads(k_cache), heads(v_cache), 128 ** -0.5, 200, 0, 4, lengths)
    attn = ops.window_fwd_bhsd(*args)
    want = R.window_attention(*args)
    assert ((attn.double() - want).abs() <= bound(want, *args[:3])).all()

    rows = attn.transpose(1, 2).reshape(B * T, H * 128)
    out = ops.mxfp4_linear(rows, *wout)
    code, byte = R.mx_quantize(rows.double().cpu())
    av, wv = R.mx_values(code, byte).to(DEV), values(*wout)
    assert ((out.double() - av @ wv.T).abs() <= product_bound(av, wv, av @ wv.T)).all()

    q8, s8, total2 = ops.rmsnorm_residual_quant(out, total, w2, 1e-6)
    want_total, y = R.rmsnorm(out, total, w2, 1e-6)
    assert torch.equal(total2, want_total)
    assert ((q8.double() * s8.double() - y).abs() <= s8.double() * (0.5 + 127 * 2 * DELTA)).all()

    w8 = torch.randint(-127, 128, (256, C), dtype=torch.int8, generator=g).to(DEV)
    cs = torch.full((256,), 1e-3, device=DEV)
    got = ops.int8_gemm_dequant(q8, s8.view(-1), w8, cs, None)
    want = (q8.double() * s8.double()) @ (w8.double() * cs.double()[:, None]).T
    # exact integer sums; the product of the scales and the scaling round to fp32, then once to bf16
    assert ((got.double() - want).abs() <= (R.BF16_HALF + 3 * 2.0 ** -24) * want.abs()).all()
    ops.check_device_status()


def block_inputs(pkg, L, hidden):
    g = torch.Generator().manual_seed(L)
    x = torch.randn((L, hidden), generator=g).to(torch.bfloat16).to(DEV)
    cos, sin = (t.to(DEV) for t in pkg.block.rope_tables(pkg.block.grid_positions(L)))
    return x, cos, sin


@pytest.mark.parametrize("window,sinks", [((100, 60), 7), ((0, 0), 0), ((-1, 0), 0)])
def test_block_with_a_window(cuda_pkg, window, sinks):
    pkg = cuda_pkg
    p = pkg.block.make_block_params(hidden=256, heads=2, ffn=512, device=DEV)
    x, cos, sin = block_inputs(pkg, 500, 256)
    taps = {}
    out = pkg.block.DiTBlock(p, window=window, sinks=sinks).forward(x, cos, sin, taps=taps)
    q, k, v = (taps["qkv"][:, i].transpose(0, 1).unsqueeze(0) for i in range(3))
    want = R.window_attention(q, k, v, 128 ** -0.5, *window, sinks)
    got = taps["attn"].view(500, 2, 128).transpose(0, 1).unsqueeze(0).double()
    assert ((got - want).abs() <= bound(want, q, k, v)).all()
    assert torch.isfinite(out.float()).all()
    assert not torch.equal(out, pkg.block.DiTBlock(p).forward(x, cos, sin))


def test_block_with_mxfp4_weights(cuda_pkg):
    """The block is its calls, bit for bit; eager, and captured and replayed."""
    pkg, ops = cuda_pkg, cuda_pkg.ops
    p = pkg.block.make_block_params(hidden=256, heads=2, ffn=512, device=DEV, weights="mxfp4")
    x, cos, sin = block_inputs(pkg, 300, 256)
    blk = pkg.block.DiTBlock(p, window=(90, 90), sinks=5)
    out = blk.forward(x, cos, sin)
    quantise = lambda t, name, q=ops.quantize_mxfp4: ops.mxfp4_gemm(*q(t), p["w4_" + name], p["s4_" + name], p["b_" + name])  # noqa: E731
    y = x.clone()
    qkv = quantise(ops.layernorm_mod(y, p["scale1"], p["shift1"]), "qkv").view(300, 3, 2, 128)
    ops.qk_norm_rope_(qkv, p["q_norm_w"], p["k_norm_w"], cos, sin)
    q, k, v = (qkv[:, i].transpose(0, 1).unsqueeze(0) for i in range(3))
    rows = ops.window_fwd_bhsd(q, k, v, 128 ** -0.5, 90, 90, 5).transpose(1, 2).reshape(300, 256)
    ops.gate_residual_(y, quantise(rows, "out"), p["gate1"])
    f = quantise(ops.layernorm_mod(y, p["scale2"], p["shift2"]), "fc1")
    ops.gate_residual_(y, quantise(f, "fc2", ops.swiglu_quantize_mxfp4), p["gate2"])
    assert torch.equal(out, y)
    graphed = pkg.block.GraphedBlock(blk, x, cos, sin)
    x2 = x.flip(0).contiguous()
    assert torch.equal(graphed(x), out) and torch.equal(graphed(x2), blk.forward(x2, cos, sin))
    with pytest.raises(ValueError, match="sinks need a window"):
        pkg.block.DiTBlock(p, sinks=3)
    with pytest.raises(ValueError, match="int8 or mxfp4"):
        pkg.block.make_block_params(hidden=256, heads=2, ffn=512, device=DEV, weights="fp8")
