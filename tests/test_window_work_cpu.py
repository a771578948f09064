"""What a windowed attention call tells the launch timer: its visible pairs' operations or its bytes,
counted in closed form, against a count over the mask."""
import random

import torch


def counted(sq, sk, left, right, sinks):
    """(visible pairs, keys that some query sees) from the mask itself."""
    p = torch.arange(sq)[:, None] + sk - sq
    j = torch.arange(sk)[None, :]
    seen = torch.ones((sq, sk), dtype=torch.bool)
    if right >= 0:
        seen &= j <= p + right
    if left >= 0:
        seen &= (j >= p - left) | (j < sinks)
    return int(seen.sum()), int(seen.any(0).sum())


CASES = [(512, 512, -1, -1, 0), (512, 512, -1, 0, 0), (512, 512, 100, 0, 4), (1, 4224, 4095, 0, 128), (836, 2000, 300, 100, 90),
         (40, 3, -1, 0, 0), (40, 3, 5, 2, 1), (7, 900, 0, 0, 900), (1, 1, 0, 0, 0), (300, 90, 30, -1, 100), (5, 64, 64, 64, 0)]
rng = random.Random(1)
CASES += [(rng.randint(1, 90), rng.randint(1, 90), rng.randint(-1, 100), rng.randint(-1, 100), rng.randint(0, 90)) for _ in range(300)]


def test_pairs_and_keys(pkg):
    for sq, sk, left, right, sinks in CASES:
        pairs, keys = counted(sq, sk, left, right, sinks)
        for b, h, hkv in ((1, 1, 1), (2, 6, 3), (1, 4096, 1)):
            bound, amount = pkg.ops._window_work(b, h, hkv, sq, sk, left, right, min(sinks, sk))
            flops, size = 4 * 128 * b * h * pairs, 2 * 128 * b * (2 * h * sq + 2 * hkv * keys)
            assert (bound, amount) == (("bf16", flops) if flops > 260 * size else ("hbm", size)), (sq, sk, left, right, sinks, h)


def test_a_causal_call_counts_half_of_a_full_one(pkg):
    full, causal = (pkg.ops._window_work(1, 24, 24, 8192, 8192, -1, right, 0) for right in (-1, 0))
    assert full == ("bf16", 4 * 128 * 24 * 8192 * 8192) and causal == ("bf16", 4 * 128 * 24 * 8192 * 8193 // 2)


def test_the_timer_takes_the_count(pkg, monkeypatch):
    """`work` is only computed for a timer, and ends up in its records."""
    class Event:
        def __init__(self, **_): pass
        def record(self, _): pass
        def synchronize(self): pass
        def elapsed_time(self, _): return 1.0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: None)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    asked = []

    def call():
        pkg.ops._call("b2_dequantize_int8_rowwise", torch.zeros(1), None, None, None, 0, 4, None,
                      work=lambda: asked.append(1) or ("hbm", 12))

    call()
    assert not asked
    with pkg.ops.LaunchTimer() as timer:
        call()
    assert timer.results() == [{"name": "b2_dequantize_int8_rowwise", "ms": 1.0, "bound": "hbm", "work": 12}]
