"""Plain 64-bit forms of the transformer-block operators, for the tests only: written from the
formulas, on whatever device the inputs are on, without the package."""
import torch

SIZES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BF16_HALF = torch.finfo(torch.bfloat16).eps / 2   # a rounding to bf16, relative


def mx_byte(largest: torch.Tensor) -> torch.Tensor:
    """Scale byte of blocks with these largest magnitudes (float64, finite)."""
    e = torch.frexp(torch.where(largest > 0, largest, 1.0))[1] - 1 - 2
    return torch.where(largest > 0, e, -127).clamp(-127, 127) + 127


def mx_elements(y: torch.Tensor, unit: torch.Tensor) -> torch.Tensor:
    """Element magnitudes 0..7 (codes) of |y| / unit: nearest, ties to the even code."""
    a = y.abs() / unit
    d = (a[..., None] - SIZES.to(y.device)).abs()
    low = d.min(-1, keepdim=True)[0]
    near = d == low                                       # one code, or two in a tie
    code = torch.arange(8, device=y.device)
    even_first = torch.where(near, code % 2 * 8 + code, 99)
    return torch.where(a >= 6, 7, even_first.min(-1)[0] % 8)


def mx_quantize(x: torch.Tensor):
    """(codes with the sign in bit 3 [M,K], scale bytes [M,K/32]) of a finite float64 matrix."""
    blocks = x.view(x.shape[0], -1, 32)
    byte = mx_byte(blocks.abs().amax(-1))
    unit = torch.exp2((byte - 127).double())[..., None]
    code = mx_elements(blocks, unit) + torch.where(torch.signbit(blocks), 8, 0)
    return code.view(x.shape), byte


def mx_codes(q: torch.Tensor) -> torch.Tensor:
    """Codes [M,K] of packed elements [M,K/2]."""
    return torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1).long()


def mx_pack(codes: torch.Tensor) -> torch.Tensor:
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8)


def mx_bytes(s: torch.Tensor, rows: int, columns: int) -> torch.Tensor:
    """Scale bytes [M,K/32] out of their tiles."""
    r = torch.arange(rows, device=s.device)[:, None]
    b = torch.arange(columns // 32, device=s.device)[None, :]
    return s[r // 128, b // 4, r % 32 * 16 + r % 128 // 32 * 4 + b % 4].long()


def mx_tiles(byte: torch.Tensor) -> torch.Tensor:
    """Tiles out of scale bytes [M,K/32]; bytes outside the matrix are 0."""
    rows, blocks = byte.shape
    s = torch.zeros((-(-rows // 128), -(-blocks // 4), 512), dtype=torch.uint8, device=byte.device)
    r = torch.arange(rows, device=s.device)[:, None]
    b = torch.arange(blocks, device=s.device)[None, :]
    s[r // 128, b // 4, r % 32 * 16 + r % 128 // 32 * 4 + b % 4] = byte.to(torch.uint8)
    return s


def mx_values(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    size = SIZES.to(codes.device)[codes & 7] * torch.where(codes >= 8, -1.0, 1.0)
    return size * torch.exp2(byte.double() - 127).repeat_interleave(32, 1)


def random_mx(rows: int, columns: int, seed: int, low: int = 120, high: int = 134):
    """A quantised matrix (packed elements, scale tiles) and its float64 values, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (rows, columns), generator=g)
    byte = torch.randint(low, high, (rows, columns // 32), generator=g)
    return mx_pack(codes), mx_tiles(byte), mx_values(codes, byte)


def rmsnorm(x: torch.Tensor, residual, weight: torch.Tensor, eps: float):
    """(sum in bf16, y in float64)."""
    total = x if residual is None else (x.double() + residual.double()).to(torch.bfloat16)
    t = total.double()
    return total, t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * weight.double()


def window_attention(q, k, v, scale, left, right, sinks=0, lengths=None):
    """float64 [B,H,Sq,D]; a query that sees no key gives zeros."""
    B, H, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    out = torch.zeros((B, H, Sq, D), dtype=torch.float64, device=q.device)
    for b in range(B):
        n = Sk if lengths is None else int(lengths[b])
        p = torch.arange(Sq, device=q.device)[:, None] + n - Sq
        j = torch.arange(n, device=q.device)[None, :]
        seen = torch.ones((Sq, n), dtype=torch.bool, device=q.device)
        if right >= 0:
            seen &= j <= p + right
        if left >= 0:
            seen &= (j >= p - left) | (j < sinks)
        rows = seen.any(1).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        for h in range(H):
            s = q[b, h, rows].double() @ k[b, h * Hkv // H, :n].double().T * scale
            w = torch.softmax(s.masked_fill(~seen[rows], float("-inf")), -1)
            # a key that a query does not see has no part in its row, whatever its value is
            vv = v[b, h * Hkv // H, :n].double()
            finite = torch.isfinite(vv)
            o = w @ torch.where(finite, vv, 0.0)
            for jj in (~finite).any(1).nonzero()[:, 0].tolist():
                see = seen[rows, jj]
                o[see] += torch.where(finite[jj], 0.0, vv[jj])
            out[b, h, rows] = o
    return out
