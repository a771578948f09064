"""The per-row bound of the windowed attention tests, without a GPU: it holds for an output with the kernel's
roundings, and no row that lost a tile, a part or an end of its keys stays within it."""
import pytest
import torch
import window_rows as W

SCALE = 128 ** -0.5


def qkv(H, Hkv, Sq, Sk, seed, spread):
    g = torch.Generator().manual_seed(seed)
    mk = lambda h, s: torch.randn(1, h, s, 128, generator=g)  # noqa: E731
    return (mk(H, Sq) * spread).bfloat16(), (mk(Hkv, Sk) * spread).bfloat16(), mk(Hkv, Sk).bfloat16()


CASES = [(2, 2, 1, 65536, -1, 0, 0, None), (3, 1, 5, 50000, 9000, 0, 3, None), (1, 1, 300, 30000, -1, 0, 0, (0, 150, 299)),
         (1, 1, 23638, 23638, 3344, 3344, 836, (0, 3000, 11819, 20000, 23637)), (2, 1, 3, 8000, -1, 0, 0, None),
         (1, 1, 2000, 109099, 3344, 3344, 836, (0, 999, 1999))]


@pytest.mark.parametrize("spread", [1.0, 2.0])
@pytest.mark.parametrize("H,Hkv,Sq,Sk,left,right,sinks,rows", CASES)
def test_lost_keys_are_seen(H, Hkv, Sq, Sk, left, right, sinks, rows, spread):
    rows = list(range(Sq)) if rows is None else list(rows)
    q, k, v = qkv(H, Hkv, Sq, Sk, Sk + Sq, spread)
    args = (q, k, v, SCALE, left, right, sinks)
    want, size = W.reference(*args, rows=rows)
    assert float(W.excess(W.rounded(*args, rows=rows), want, size, q, k, SCALE).max()) < 1.0
    if spread > 1:                                          # a few keys have the weight: most tiles hold nothing
        return
    p = [r + Sk - Sq for r in rows]
    for i, at in enumerate(p):
        first, last = max(at - left, 0) if left >= 0 else 0, min(at + right, Sk - 1) if right >= 0 else Sk - 1
        middle = (first + last) // 2
        lost = {"a tile in the middle": (middle, middle + 128), "the last tile": (last - 127, last + 1), "the first tile": (first, first + 128),
                "an eighth": (first + (last - first) // 8, first + (last - first) // 4)}
        if sinks and first >= sinks:
            lost["a first tile that stays visible"] = (0, min(128, sinks))
        for what, drop in lost.items():
            got, _ = W.reference(*args, rows=rows[i:i + 1], drop=(max(drop[0], 0), drop[1]))
            if what.startswith("a first") and sinks < 100:  # some three keys of thousands: not in every row
                continue
            over = W.excess(got.bfloat16(), want[:, :, i:i + 1], size[:, :, i:i + 1], q, k, SCALE)
            assert bool((over > 1).all()), (what, at, float(over.min()))


def test_rows_without_keys():
    q, k, v = qkv(1, 1, 6, 3, 1, 1.0)
    want, size = W.reference(q, k, v, SCALE, -1, 0)
    assert not want[0, 0, :3].any() and not size[0, 0, :3].any()
    got = want.bfloat16()
    assert float(W.excess(got, want, size, q, k, SCALE).max()) < 1
    got[0, 0, 1, 5] = 1e-8
    assert float(W.excess(got, want, size, q, k, SCALE).max()) > 1
