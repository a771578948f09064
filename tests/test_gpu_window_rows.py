"""Windowed attention, row by row: a bound that shrinks with the number of keys, so that a lost or doubled tile,
part or split boundary shows at every length; and the calls that leave their parts in memory, on two
streams at once and in two graphs."""
import pytest
import torch
import window_rows as W

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 128 ** -0.5


def qkv(B, H, Hkv, Sq, Sk, seed, spread):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda h, s, a: (torch.randn((B, s, h, 128), generator=g, device=DEV) * a).to(torch.bfloat16).transpose(1, 2)  # noqa: E731
    return mk(H, Sq, spread), mk(Hkv, Sk, spread), mk(Hkv, Sk, 1.0)


def some_rows(Sq, most=96):
    """All rows, or those at the ends, in the middle, at tile borders and spread out."""
    if Sq <= most:
        return list(range(Sq))
    pick = set(range(12)) | set(range(Sq - 12, Sq)) | set(range(Sq // 2 - 6, Sq // 2 + 6))
    pick |= {i * Sq // 40 for i in range(40)} | {x for x in (127, 128, 255, 256, 257) if x < Sq}
    return sorted(pick)


def check(pkg, q, k, v, left, right, sinks=0, lengths=None):
    got = pkg.ops.window_fwd_bhsd(q, k, v, SCALE, left, right, sinks, lengths)
    rows = some_rows(q.shape[2])
    want, spread = W.reference(q, k, v, SCALE, left, right, sinks, lengths, rows=rows)
    over = W.excess(got[:, :, rows], want, spread, q, k, SCALE)
    assert bool((over <= 1).all()), (float(over.max()), int((over > 1).sum()), (over > 1).nonzero()[:4].tolist())
    pkg.ops.check_device_status()
    return got


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (0, 0, 5), (127, 128, 0), (200, 0, 4), (300, 40, 130), (5, 900, 700), (-1, 7, 3), (90, -1, 3)]


@pytest.mark.parametrize("spread", [1.0, 2.0])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk", [(2, 3, 3, 129, 129), (1, 4, 2, 513, 513), (1, 6, 2, 700, 700), (3, 8, 2, 1, 1000), (1, 24, 1, 5, 333),
                                           (2, 4, 4, 17, 2050), (1, 3, 3, 200, 1500), (1, 2, 1, 300, 4000), (1, 2, 2, 700, 90)])
def test_sizes_and_windows(cuda_pkg, B, H, Hkv, Sq, Sk, left, right, sinks, spread):
    check(cuda_pkg, *qkv(B, H, Hkv, Sq, Sk, Sq + Sk, spread), left, right, sinks)


@pytest.mark.parametrize("spread", [1.0, 2.0])
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,memory", [(1, 2, 2, 1, 65536, True), (1, 3, 1, 40, 50000, True), (1, 24, 24, 836, 9000, True),
                                                  (1, 1, 1, 300, 30000, True), (1, 24, 24, 836, 24244, True), (1, 24, 24, 1, 8192, False),
                                                  (1, 24, 6, 3, 8000, False), (1, 8, 8, 256, 2000, False), (8, 24, 6, 1, 16411, False)])
def test_parts_of_long_key_sequences(cuda_pkg, B, H, Hkv, Sq, Sk, memory, spread):
    assert (cuda_pkg.ops._window_workspace(B, H, Hkv, Sq, Sk, -1, 0, 0) > 0) == memory
    q, k, v = qkv(B, H, Hkv, Sq, Sk, Sk, spread)
    check(cuda_pkg, q, k, v, -1, 0)
    check(cuda_pkg, q, k, v, 9000, 0, 3)
    check(cuda_pkg, q, k, v, 4095, 100, 836)
    lengths = torch.randint(1, Sk + 1, (B,), generator=torch.Generator().manual_seed(Sk), dtype=torch.int32).to(DEV)
    check(cuda_pkg, q, k, v, -1, 0, 0, lengths)
    check(cuda_pkg, q, k, v, 2000, 0, 130, lengths)


@pytest.mark.parametrize("S,H,Hkv,left,right,sinks", [(23638, 3, 3, 3344, 3344, 836), (40000, 2, 1, 1023, 0, 4), (30000, 1, 1, -1, 0, 0),
                                                      (109099, 2, 2, 3344, 3344, 836), (109099, 1, 1, -1, 3344, 0)])
def test_long_sequences(cuda_pkg, S, H, Hkv, left, right, sinks):
    check(cuda_pkg, *qkv(1, H, Hkv, S, S, S % 1000, 1.0), left, right, sinks)


MEMORY = [(1, 2, 2, 1, 65536), (1, 3, 1, 40, 50000), (1, 24, 24, 836, 9000), (1, 1, 1, 300, 30000)]


@pytest.mark.parametrize("B,H,Hkv,Sq,Sk", MEMORY)
def test_parts_in_memory_on_two_streams_at_once(cuda_pkg, B, H, Hkv, Sq, Sk):
    """Calls alternate between two streams without waiting for one another: the bits of the same calls
    one after the other."""
    ops = cuda_pkg.ops
    assert ops._window_workspace(B, H, Hkv, Sq, Sk, -1, 0, 0) > 0
    _, k, v = qkv(B, H, Hkv, 1, Sk, 5, 1.0)
    qs = [qkv(B, H, Hkv, Sq, 1, 10 + i, 1.0)[0] for i in range(6)]
    want = [ops.window_fwd_bhsd(q, k, v, SCALE, -1, 0) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)]
    got = []
    for turn in range(8):
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[(i + turn) % 2]):
                got.append((i, ops.window_fwd_bhsd(q, k, v, SCALE, -1, 0)))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for i, out in got)
    ops.check_device_status()


@pytest.mark.parametrize("B,H,Hkv,Sq,Sk", MEMORY[:3])
def test_parts_in_memory_in_two_graphs(cuda_pkg, B, H, Hkv, Sq, Sk):
    """Two captures of the call, replayed in turn and at once on two streams, on inputs that change."""
    ops = cuda_pkg.ops
    _, k, v = qkv(B, H, Hkv, 1, Sk, 5, 1.0)
    qs = [qkv(B, H, Hkv, Sq, 1, 20 + i, 1.0)[0].contiguous() for i in range(4)]
    want = [ops.window_fwd_bhsd(q, k, v, SCALE, -1, 0).clone() for q in qs]
    static = [qs[0].clone(), qs[1].clone()]
    graphs, outs, streams = [], [], [torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)]
    for q in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.window_fwd_bhsd(q, k, v, SCALE, -1, 0))
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1):
            static[i].copy_(qs[(turn + i) % 4])
        torch.cuda.synchronize()
        for _ in range(3):
            for i in (0, 1):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(outs[i], want[(turn + i) % 4])
    ops.check_device_status()


def test_the_timer_counts_visible_pairs(cuda_pkg):
    q, k, v = qkv(1, 4, 4, 1000, 1000, 1, 1.0)
    with cuda_pkg.ops.LaunchTimer() as timer:
        cuda_pkg.ops.window_fwd_bhsd(q, k, v, SCALE, -1, -1)
        cuda_pkg.ops.window_fwd_bhsd(q, k, v, SCALE, -1, 0)
        cuda_pkg.ops.window_fwd_bhsd(q[:, :, :1], k, v, SCALE, 99, 0, 7)
    full, causal, token = timer.results()
    assert (full["bound"], full["work"]) == ("bf16", 4 * 128 * 4 * 1000 * 1000)
    # half of the operations, and the same 4 MB: 250 operations per byte
    assert (causal["bound"], causal["work"]) == ("hbm", 2 * 128 * 4 * 1000 * 4)
    assert (token["bound"], token["work"]) == ("hbm", 2 * 128 * (2 * 4 + 2 * 4 * 107))
