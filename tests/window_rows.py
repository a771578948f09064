"""Rows of windowed attention in 64 bits with a bound that shrinks as a row's keys grow in number, for the
tests only."""
import torch

HALF = torch.finfo(torch.bfloat16).eps / 2


def reference(q, k, v, scale, left, right, sinks=0, lengths=None, rows=None, drop=None):
    """(want, spread) of the given query rows, float64: the output [B,H,rows,D] and
    sqrt(sum over the keys of weight^2 |v|^2) [B,H,rows,1].  `drop` = (first, last): keys left out."""
    B, H, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    rows = torch.arange(Sq) if rows is None else torch.as_tensor(rows)
    rows = rows.to(q.device)
    want = torch.zeros((B, H, rows.numel(), D), dtype=torch.float64, device=q.device)
    spread = torch.zeros((B, H, rows.numel(), 1), dtype=torch.float64, device=q.device)
    for b in range(B):
        n = Sk if lengths is None else int(lengths[b])
        p = rows[:, None] + n - Sq
        j = torch.arange(n, device=q.device)[None, :]
        seen = torch.ones((rows.numel(), n), dtype=torch.bool, device=q.device)
        if right >= 0:
            seen &= j <= p + right
        if left >= 0:
            seen &= (j >= p - left) | (j < sinks)
        if drop is not None:
            seen[:, drop[0]:drop[1]] = False
        some = seen.any(1, keepdim=True)
        for h in range(H):
            kk, vv = k[b, h * Hkv // H, :n].double(), v[b, h * Hkv // H, :n].double()
            s = (q[b, h, rows].double() @ kk.T * scale).masked_fill(~seen, float("-inf"))
            w = torch.softmax(torch.where(some, s, 0.0), -1) * some
            want[b, h] = w @ vv
            spread[b, h] = ((w * w) @ (vv * vv).sum(1, keepdim=True)).sqrt()
    return want, spread


def limit(want, spread, q, k, scale):
    """How far a row's output may be off, as the norm over its D columns.  Every weight is rounded to bf16,
    a relative error of at most HALF that has nothing to do with the values, so the errors of a row's
    keys add up like independent ones: HALF * spread at most (their own root mean square is below
    HALF / sqrt(3); the norm over 128 columns stays within a few per cent of it).  The output is rounded
    once.  Exponentials (1e-4) and scores (ten roundings of 2^-23 of the largest sum of magnitudes) move a
    row's weights less than their rounding does, and add to it."""
    norm = lambda t: t.double().norm(dim=-1).amax()  # noqa: E731
    weight = HALF + 1e-4 + 2 * 10 * 2.0 ** -23 * scale * norm(q) * norm(k)
    return weight * spread + HALF * want.norm(dim=-1, keepdim=True)


def excess(got, want, spread, q, k, scale):
    """The largest ratio of a row's error to its limit; a row that sees nothing has to be zeros."""
    err = (got.double() - want).norm(dim=-1, keepdim=True)
    most = limit(want, spread, q, k, scale)
    return torch.where(most > 0, err / most.clamp(min=1e-300), torch.where(err > 0, 9e9, 0.0))


def rounded(q, k, v, scale, left, right, sinks=0, lengths=None, rows=None):
    """The output with the kernel's two roundings: weights (of the row's largest) and result in bf16."""
    B, H, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    rows = torch.arange(Sq) if rows is None else torch.as_tensor(rows)
    out = torch.zeros((B, H, rows.numel(), D), dtype=torch.bfloat16)
    for b in range(B):
        n = Sk if lengths is None else int(lengths[b])
        p = rows[:, None] + n - Sq
        j = torch.arange(n)[None, :]
        seen = torch.ones((rows.numel(), n), dtype=torch.bool)
        if right >= 0:
            seen &= j <= p + right
        if left >= 0:
            seen &= (j >= p - left) | (j < sinks)
        for h in range(H):
            s = (q[b, h, rows].double() @ k[b, h * Hkv // H, :n].double().T * scale).masked_fill(~seen, float("-inf"))
            e = torch.exp(s - s.amax(1, keepdim=True).clamp(min=-1e300))
            out[b, h] = (e.to(torch.bfloat16).double() @ v[b, h * Hkv // H, :n].double() / e.sum(1, keepdim=True).clamp(min=1e-300)).to(torch.bfloat16)
    return out
