"""The transformer-block operators next to one another on two streams at once, and in graphs that are replayed
at once: the bits of the same calls one after the other."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def calls(pkg):
    ops = pkg.ops
    g = torch.Generator(device=DEV).manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    x, r, w = rnd(2000, 1536), rnd(2000, 1536), rnd(1536)
    odd = rnd(300, 1001)
    wide = rnd(900, 2048)
    a, weights, few = ops.quantize_mxfp4(rnd(1500, 1024)), ops.quantize_mxfp4(rnd(2304, 1024)), ops.quantize_mxfp4(rnd(5, 1024))
    bias = rnd(2304)
    q, k, v = (rnd(1, 900, 6, 128).transpose(1, 2) for _ in range(3))
    token, cache_k, cache_v = rnd(2, 1, 6, 128).transpose(1, 2), rnd(2, 3000, 2, 128).transpose(1, 2), rnd(2, 3000, 2, 128).transpose(1, 2)
    long_q, long_k, long_v = rnd(1, 40, 3, 128).transpose(1, 2), rnd(1, 50000, 1, 128).transpose(1, 2), rnd(1, 50000, 1, 128).transpose(1, 2)
    return [lambda: ops.rmsnorm_residual_quant(x, r, w), lambda: ops.rmsnorm_residual_mxfp4(x, r, w), lambda: ops.rmsnorm_residual_quant(odd, None, odd[0].clone()),
            lambda: ops.quantize_mxfp4(wide), lambda: ops.swiglu_quantize_mxfp4(wide), lambda: ops.dequantize_mxfp4(*a),
            lambda: ops.mxfp4_gemm(*a, *weights, bias), lambda: ops.mxfp4_gemm(*few, *weights, bias), lambda: ops.mxfp4_linear(wide[:, :1024].contiguous(), *weights),
            lambda: ops.window_fwd_bhsd(q, k, v, 0.1, 100, 20, 5), lambda: ops.window_fwd_bhsd(token, cache_k, cache_v, 0.1, 2000, 0, 4),
            lambda: ops.window_fwd_bhsd(long_q, long_k, long_v, 0.1, -1, 0), lambda: ops.fwd_bhsd(q, k, v, 0.1)]


def bits(out):
    return [t.contiguous().view(torch.uint8) for t in (out if isinstance(out, (list, tuple)) else [out])]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(bits(a), bits(b)))


def test_all_pairs_at_once(cuda_pkg):
    fs = calls(cuda_pkg)
    want = [f() for f in fs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)]
    for shift in range(len(fs)):
        got = []
        for i in range(len(fs)):
            for s, j in ((0, i), (1, (i + shift) % len(fs))):
                with torch.cuda.stream(streams[s]):
                    got.append((j, fs[j]()))
        torch.cuda.synchronize()
        assert all(same(out, want[j]) for j, out in got)
    cuda_pkg.ops.check_device_status()


def test_graphs_replayed_at_once(cuda_pkg):
    fs = calls(cuda_pkg)
    want = [f() for f in fs]
    graphs = []
    for order in (range(len(fs)), reversed(range(len(fs)))):
        graph, outs = torch.cuda.CUDAGraph(), {}
        with torch.cuda.graph(graph):
            for i in order:
                outs[i] = fs[i]()
        graphs.append((graph, outs))
    streams = [torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)]
    for _ in range(5):
        for _, outs in graphs:                              # what a replay leaves out would stay zero
            for i, out in outs.items():
                for t in (out if isinstance(out, (list, tuple)) else [out])[:2]:   # the third is the norm's sum: x itself without a residual
                    t.zero_()
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(same(outs[i], want[i]) for _, outs in graphs for i in outs)
    cuda_pkg.ops.check_device_status()
