"""Attention with a sliding window and first keys that stay visible, against a plain 64-bit form."""
import operator_refs as R
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 128 ** -0.5


def qkv(B, H, Hkv, Sq, Sk, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda h, s: (torch.randn(B, s, h, 128, generator=g) * spread).to(torch.bfloat16).to(DEV).transpose(1, 2)  # noqa: E731
    return mk(H, Sq), mk(Hkv, Sk), mk(Hkv, Sk)


def bound(want, q, k, v, scale=SCALE):
    """A weight is off by its rounding to bf16 (half a step), its exponential (1e-4 at most) and its
    score: ten roundings of 2^-23 (eight matrix instructions of 16 products, scaling, subtracting
    the maximum) of the largest possible sum of magnitudes, once in the weight and once in their
    sum.  That times the largest |V|, and the output is rounded once."""
    norm = lambda t: t.double().nan_to_num(0, 0, 0).norm(dim=-1).amax()  # noqa: E731
    big = v.double().nan_to_num(0, 0, 0).abs().amax()
    score = 2 * 10 * 2.0 ** -23 * scale * norm(q) * norm(k)
    return (R.BF16_HALF + 1e-4 + score) * big + R.BF16_HALF * want.abs()


def check(pkg, q, k, v, left, right, sinks=0, lengths=None, scale=SCALE):
    got = pkg.ops.window_fwd_bhsd(q, k, v, scale, left, right, sinks, lengths)
    again = pkg.ops.window_fwd_bhsd(q, k, v, scale, left, right, sinks, lengths)
    pkg.ops.check_device_status()
    want = R.window_attention(q, k, v, scale, left, right, sinks, lengths)
    assert got.shape == q.shape and got.transpose(1, 2).is_contiguous()
    # NaN and infinities have to be where the formula has them, the rest within the bound
    same = (got.double() == want) | (got.isnan() & want.isnan())
    err = torch.where(same, 0.0, (got.double() - want).abs())
    fine = same | (torch.isfinite(want) & (err <= bound(want, q, k, v, scale)))
    assert bool(fine.all()), (float(err.nan_to_num(9e9).max()), int((~fine).sum()))
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))   # deterministic
    return got


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (0, 0, 0), (0, 0, 5), (63, 0, 0), (127, 128, 0), (200, 0, 4), (300, 40, 130), (5, 900, 700), (-1, 7, 3)]


@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("B,H,Hkv,S", [(1, 1, 1, 1), (1, 2, 2, 127), (2, 3, 3, 129), (1, 4, 2, 513), (1, 6, 2, 700)])
def test_self_attention(cuda_pkg, B, H, Hkv, S, left, right, sinks):
    check(cuda_pkg, *qkv(B, H, Hkv, S, S, S), left, right, sinks)


@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk", [(1, 1, 1, 1, 128), (3, 8, 2, 1, 1000), (1, 24, 1, 5, 333), (2, 4, 4, 17, 2050),
                                           (1, 3, 3, 200, 1500), (1, 2, 1, 300, 4000), (1, 2, 2, 700, 90), (2, 2, 1, 40, 3)])
def test_queries_at_the_end_of_a_cache(cuda_pkg, B, H, Hkv, Sq, Sk, left, right, sinks):
    """More keys than queries, and fewer: then the first queries see nothing (or nothing but what
    `right` lets them see)."""
    check(cuda_pkg, *qkv(B, H, Hkv, Sq, Sk, Sq + Sk), left, right, sinks)


@pytest.mark.parametrize("left,right,sinks", [(-1, -1, 0), (100, 0, 4), (-1, 0, 0), (300, 20, 200)])
@pytest.mark.parametrize("Sq", [1, 7, 260])
def test_lengths_and_what_lies_behind_them(cuda_pkg, Sq, left, right, sinks):
    """Sequences from no key to all, on the device; the cache behind them holds NaN and infinities."""
    B, H, Hkv, Sk = 7, 4, 2, 900
    q, k, v = qkv(B, H, Hkv, Sq, Sk, Sq)
    lengths = torch.tensor([0, 1, 5, 128, 555, 899, 900], dtype=torch.int32, device=DEV)
    for b, n in enumerate(lengths.tolist()):
        k[b, :, n:] = float("nan")
        v[b, :, n:] = float("inf")
        v[b, :, n:, ::3] = float("nan")
    got = check(cuda_pkg, q, k, v, left, right, sinks, lengths)
    assert not got[0].any() and torch.isfinite(got.float()).all()
    # out of range: clamped
    wild = torch.tensor([-3, 1, 5, 128, 555, 899, 1 << 30], dtype=torch.int32, device=DEV)
    assert torch.equal(cuda_pkg.ops.window_fwd_bhsd(q, k, v, SCALE, left, right, sinks, wild), got)


@pytest.mark.parametrize("Sq,Sk", [(1, 700), (3, 700), (700, 700), (300, 2000)])
def test_non_finite_values_reach_only_who_sees_them(cuda_pkg, Sq, Sk):
    q, k, v = qkv(1, 2, 2, Sq, Sk, 3)
    for j, x in [(0, float("inf")), (5, float("nan")), (130, float("-inf")), (Sk - 400, float("nan")), (Sk - 130, float("inf")), (Sk - 1, float("inf"))]:
        v[0, 0, j, j % 128] = x
        k[0, 1, j] = float("nan")
    for window in [(20, 0, 3), (127, 127, 0), (0, 0, 0), (100, 30, 140)]:
        got = check(cuda_pkg, q, k, v, *window)
        if Sq == 700:
            assert torch.isfinite(got.float()).any() and not torch.isfinite(got.float()).all()


def test_large_scores_and_infinite_ones(cuda_pkg):
    """Rows whose maximum grows late and far, and scores of minus infinity."""
    q, k, v = qkv(1, 2, 1, 300, 900, 5, 4.0)
    k[0, 0, 500:] *= 8.0
    check(cuda_pkg, q, k, v, -1, 0)
    check(cuda_pkg, q, k, v, 400, 100, 10)
    check(cuda_pkg, q[:, :, :2], k, v, -1, 0)
    q = q.abs() + 0.1
    k[0, 0, 100:200] = float("-inf")                            # scores -inf: weight 0
    check(cuda_pkg, q, k, v, -1, -1)
    check(cuda_pkg, q[:, :, :1].contiguous(), k, v, 30, 0, 200)
    k[0, 0, :] = float("-inf")                                  # 0 / 0, as the formula has it
    assert cuda_pkg.ops.window_fwd_bhsd(q, k, v, SCALE, -1, 0).isnan().all()
    assert cuda_pkg.ops.window_fwd_bhsd(q[:, :, :1], k, v, SCALE, -1, 0).isnan().all()


@pytest.mark.parametrize("Sq,Sk", [(333, 333), (2, 333), (1, 40)])
def test_strides_and_orders(cuda_pkg, Sq, Sk):
    """Packed projections, head-major caches, slices with gaps: the bits of contiguous tensors."""
    g = torch.Generator().manual_seed(9)
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV)  # noqa: E731
    packed = rnd(2, Sk, 3, 4, 128)
    q, k, v = (packed[:, :, i].transpose(1, 2) for i in range(3))
    q = q[:, :, -Sq:]
    wide = rnd(2, 4, Sk, 320)
    cases = [(q, k, v), (q, k.contiguous(), v.contiguous()), (q.contiguous(), wide[..., 64:192], wide[..., 192:]),
             (q[:, :, :, :], rnd(Sk, 4, 2, 128).permute(2, 1, 0, 3), rnd(4, Sk, 2, 128).permute(2, 0, 1, 3)),
             (q[:1], k[:1, :1], v[1:, :1])]
    for q, k, v in cases:
        for window in [(100, 0, 4), (50, 60, 0)]:
            a = cuda_pkg.ops.window_fwd_bhsd(q, k, v, SCALE, *window)
            b = cuda_pkg.ops.window_fwd_bhsd(q.contiguous(), k.contiguous(), v.contiguous(), SCALE, *window)
            assert torch.equal(a, b)
            check(cuda_pkg, q, k, v, *window)


def test_whole_window_is_the_full_attention(cuda_pkg):
    """Without limits: the full kernel's result.  The key sequence may be split over CTAs here, which
    sums in another order, so each is held to its own bound."""
    q, k, v = qkv(1, 3, 3, 1300, 1300, 2)
    full = cuda_pkg.ops.fwd_bhsd(q, k, v, SCALE).double()
    for limit in (-1, 1 << 60):
        got = cuda_pkg.ops.window_fwd_bhsd(q, k, v, SCALE, limit, limit).double()
        assert ((got - full).abs() <= 2 * bound(full, q, k, v)).all()


@pytest.mark.parametrize("S,H,left,right,sinks", [(23638, 2, 3344, 3344, 836), (40000, 1, 1023, 0, 4)])
def test_long_sequences_sampled_rows(cuda_pkg, S, H, left, right, sinks):
    q, k, v = qkv(1, H, H, S, S, 11)
    got = cuda_pkg.ops.window_fwd_bhsd(q, k, v, SCALE, left, right, sinks)
    cuda_pkg.ops.check_device_status()
    assert torch.isfinite(got.float()).all()
    for r0 in (0, S // 2, S - 300):
        # rows r0.. of the sequence as the end of a shorter one, with `right` keys behind them in sight
        rows = torch.arange(r0, r0 + 300, device=DEV)
        j = torch.arange(S, device=DEV)
        seen = (j <= rows[:, None] + right) & ((j >= rows[:, None] - left) | (j < sinks))
        s = (q[0, :, rows].double() @ k[0].double().transpose(-1, -2) * SCALE).masked_fill(~seen, float("-inf"))
        want = torch.softmax(s, -1) @ v[0].double()
        assert ((got[0, :, rows].double() - want).abs() <= bound(want, q, k, v)).all()


def test_long_cache_offsets_past_32_bits(cuda_pkg):
    """A cache of more than 2^31 elements: single tokens and a chunk at its end."""
    Sk, Hkv = 262144 + 77, 70
    assert Sk * Hkv * 128 > 2 ** 31
    k = torch.zeros((1, Sk, Hkv, 128), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    g = torch.Generator(device=DEV).manual_seed(4)
    k[:, -1500:] = torch.randn((1, 1500, Hkv, 128), device=DEV, generator=g).to(torch.bfloat16)
    v[:, -1500:] = torch.randn((1, 1500, Hkv, 128), device=DEV, generator=g).to(torch.bfloat16)
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    for Sq in (1, 150):
        q = torch.randn((1, Hkv, Sq, 128), device=DEV, generator=g).to(torch.bfloat16)
        a = cuda_pkg.ops.window_fwd_bhsd(q, k, v, SCALE, 1000, 0, 0)
        want = R.window_attention(q[:, -3:], k[:, -3:, -1300:], v[:, -3:, -1300:], SCALE, 1000, 0)
        assert ((a[:, -3:].double() - want).abs() <= bound(want, q, k[:, -3:, -1300:], v[:, -3:, -1300:])).all()


@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,memory", [(1, 2, 2, 1, 65536, True), (1, 3, 1, 40, 50000, True), (1, 24, 24, 836, 9000, True),
                                                  (1, 1, 1, 300, 30000, True), (1, 24, 24, 1, 8192, False),
                                                  (1, 24, 6, 3, 8000, False), (1, 8, 8, 256, 2000, False)])
def test_every_way_to_join_the_parts(cuda_pkg, B, H, Hkv, Sq, Sk, memory):
    """Key sequences split over a cluster, or through memory, by few rows and by whole tiles."""
    need = cuda_pkg.ops._window_workspace(B, H, Hkv, Sq, Sk, -1, 0, 0)
    assert (need > 0) == memory
    q, k, v = qkv(B, H, Hkv, Sq, Sk, 17)
    check(cuda_pkg, q, k, v, -1, 0)
    check(cuda_pkg, q, k, v, 9000, 0, 3)
    lengths = torch.full((B,), Sk * 2 // 3, dtype=torch.int32, device=DEV)
    check(cuda_pkg, q, k, v, -1, 0, 0, lengths)
    check(cuda_pkg, q, k, v, -1, 5, 0, lengths * 0 + 100)            # most parts have nothing to do


def test_side_stream_two_captures_and_lengths_that_change(cuda_pkg):
    """Single tokens captured twice in graphs that are replayed in turn while the lengths grow."""
    ops = cuda_pkg.ops
    q, k, v = qkv(3, 8, 2, 1, 2000, 8)
    q2 = q.flip(0).contiguous()
    lengths = torch.tensor([40, 700, 1990], dtype=torch.int32, device=DEV)
    ops.window_fwd_bhsd(q, k, v, SCALE, 500, 0, 4, lengths)
    graphs = []
    for x in (q, q2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.window_fwd_bhsd(x, k, v, SCALE, 500, 0, 4, lengths)
        graphs.append((graph, x, out))
    for _ in range(3):
        lengths += 3
        for graph, _, _ in graphs:
            graph.replay()
        for _, x, out in graphs:
            assert torch.equal(out, ops.window_fwd_bhsd(x, k, v, SCALE, 500, 0, 4, lengths))
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.window_fwd_bhsd(q, k, v, SCALE, 500, 0, 4, lengths)
    b = ops.window_fwd_bhsd(q, k, v, SCALE, 500, 0, 4, lengths)      # at the same time on another
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def test_refusals(cuda_pkg):
    ops = cuda_pkg.ops
    q, k, v = qkv(1, 4, 2, 16, 32, 1)
    f = ops.window_fwd_bhsd
    for call, match in [(lambda: f(q.half(), k, v, SCALE, 1, 1), "BF16"),
                        (lambda: f(q, k.half(), v, SCALE, 1, 1), "same dtype"),
                        (lambda: f(q, k, v[:, :1], SCALE, 1, 1), "same shape"),
                        (lambda: f(q[..., :64], k[..., :64], v[..., :64], SCALE, 1, 1), "head dimension 128"),
                        (lambda: f(q[:, :3], k, v, SCALE, 1, 1), "multiple of the key heads"),
                        (lambda: f(q[:, :, :0], k, v, SCALE, 1, 1), "must be positive"),
                        (lambda: f(q, k, v, 0.0, 1, 1), "finite and positive"),
                        (lambda: f(q, k, v, SCALE, -2, 1), "at least -1"),
                        (lambda: f(q, k, v, SCALE, 1, 1, -1), "at least -1"),
                        (lambda: f(q, k, v, SCALE, 1, 1, 0, torch.zeros(2, dtype=torch.int32, device=DEV)), "kv_lengths"),
                        (lambda: f(q, k, v, SCALE, 1, 1, 0, torch.zeros(1, dtype=torch.int64, device=DEV)), "kv_lengths"),
                        (lambda: f(q, k.cpu(), v, SCALE, 1, 1), "CUDA device"),
                        (lambda: f(q, k[:, :1].expand(1, 2, 32, 128), v, SCALE, 1, 1), "strides must be positive"),
                        (lambda: f(q, torch.zeros((1, 2, 32, 132), dtype=torch.bfloat16, device=DEV)[..., :128], v, SCALE, 1, 1), "multiples of 8"),
                        (lambda: f(q, torch.zeros((1, 2, 128, 32), dtype=torch.bfloat16, device=DEV).transpose(2, 3), v, SCALE, 1, 1), "contiguous last")]:
        with pytest.raises(RuntimeError, match=match):
            call()


@pytest.mark.parametrize("B,H,Hkv", [(5, 27, 27), (5, 33, 11), (7, 39, 13)])
def test_more_items_than_one_order_of_positions(cuda_pkg, B, H, Hkv):
    """Row groups enough for two orders of positions one after the other and for three, the last of them
    with fewer groups (of one head, of three)."""
    q, k, v = qkv(B, H, Hkv, 2100, 2100, H)
    lengths = torch.tensor([2100, 37, 1500, 0, 2099, 2100, 700], dtype=torch.int32, device=DEV)[:B].contiguous()
    check(cuda_pkg, q, k, v, 130, 0, 4)
    check(cuda_pkg, q, k, v, 130, 0, 4, lengths)


@pytest.mark.parametrize("B,H,Hkv,Sq,Sk", [(1, 2, 2, 700, 700), (2, 6, 2, 1100, 900), (1, 4, 1, 3, 600), (2, 31, 31, 1300, 1300)])
@pytest.mark.parametrize("left,sinks", [(0, 0), (100, 3), (500, 0)])
def test_a_limit_behind_and_none_ahead(cuda_pkg, B, H, Hkv, Sq, Sk, left, sinks):
    """The first positions see the most keys."""
    q, k, v = qkv(B, H, Hkv, Sq, Sk, Sq + left)
    check(cuda_pkg, q, k, v, left, -1, sinks)
    check(cuda_pkg, q, k, v, left, -1, sinks, torch.tensor([Sk // 3, Sk], dtype=torch.int32, device=DEV)[:B].contiguous())
