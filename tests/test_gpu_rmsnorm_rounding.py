"""The norm's roundings, on rows whose sum of squares is exact: mean, 1 / sqrt, scale = max|y| / 127 and
y / scale are each one correctly rounded fp32 operation, and q the whole number next to the last."""
import operator_refs as R
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def exact_rows(m, c, seed):
    """bf16 rows of whole numbers up to 181 with a mean square of 64^2: in groups of eight, one that the
    whole row shares, three random ones and four whose squares fill up to 8 * 64^2; 64 behind the
    last group.  Every partial sum stays below 2^24, so the multiplier is 1/64 exactly, in any order
    of the additions, and y = x * weight / 64 has at most 16 bits."""
    assert c * 4096 < 1 << 24
    g = torch.Generator().manual_seed(seed)
    i = torch.arange(182)
    sums = (i[:, None, None] ** 2 + i[None, :, None] ** 2 + i[None, None, :] ** 2).flatten()
    three = torch.full((32769,), -1)                        # a number that is three squares -> where it was found
    three[sums[sums <= 32768]] = torch.arange(sums.numel())[sums <= 32768]
    groups = m * (c // 8)
    x = torch.randint(-90, 91, (groups, 8), generator=g)
    x[:, 0] = (torch.randint(23, 91, (m,), generator=g) * 2 + 1).repeat_interleave(c // 8)
    x[:, 1:4] = torch.where((x[:, :4] ** 2).sum(1, keepdim=True) > 32000, 0, x[:, 1:4])
    left = 32768 - (x[:, :4] ** 2).sum(1)
    fourth = torch.zeros(groups, dtype=torch.int64)
    for d in range(1, 9):
        fourth = torch.where((three[left - fourth ** 2] < 0) & (left >= d * d), d, fourth)
    at = three[left - fourth ** 2]
    assert (at >= 0).all()
    x[:, 4:] = torch.stack((fourth, at // (182 * 182), at // 182 % 182, at % 182), 1)
    x *= torch.where(torch.rand(x.shape, generator=g) < 0.5, -1, 1)
    x = torch.cat((x.view(m, -1), torch.full((m, c % 8), 64)), 1)
    assert ((x * x).sum(1) == c * 4096).all()
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("top", [127, 101])
@pytest.mark.parametrize("c", [41, 392, 984, 1001, 2047, 3080, 4088])
def test_scale_and_elements_are_divisions(cuda_pkg, c, top):
    """Widths of the vector kernel and of the odd one; in one run the pointers start off a vector."""
    m = 600
    x = exact_rows(m, c, c)
    # the row's shared value makes the maximum, `top` times it, and with 127 exact ties, (k + 1/2) times it
    g = torch.Generator().manual_seed(c)
    w = torch.rand(c, generator=g) * 0.5
    w[:c // 8 * 8:8] = torch.randint(0, top, (c // 8,), generator=g) + 0.5
    w[0] = top
    w = w.to(torch.bfloat16)
    y = x.float() * w.float() / 64                          # exact
    # on the CPU: on a GPU torch multiplies by the reciprocal of a divisor that is a number
    want_s = (y.abs().amax(1, keepdim=True) / 127.0).clamp(min=1e-30)
    want_q = (y / want_s).round()
    shifted = torch.empty(m * c + 3, dtype=torch.bfloat16, device=DEV)[3:].view(m, c).copy_(x)
    for rows in (x.to(DEV), shifted):
        q, s, _ = (t.cpu() for t in cuda_pkg.ops.rmsnorm_residual_quant(rows, None, w.to(DEV), 0.0))
        assert torch.equal(s, want_s), int((s != want_s).sum())
        assert torch.equal(q.float(), want_q), int((q.float() != want_q).sum())


def rounded_norm(x, w, eps):
    """y in fp32 of rows of small whole numbers (the sum of squares is exact in any order), every step
    rounded once: mean, its sum with eps, 1 / sqrt, times x, times the weight."""
    total = (x.long() ** 2).sum(1, keepdim=True)
    assert int(total.max()) < 1 << 24
    mean = total.float() / torch.tensor(float(x.shape[1])) + torch.tensor(eps)
    rstd = (1.0 / torch.sqrt(mean.double())).float()
    return x.float() * rstd * w.float()


@pytest.mark.parametrize("eps", [0.0, 1e-6, 0.3])
@pytest.mark.parametrize("c", [32, 37, 416, 1001, 1312, 4096, 16384])
def test_every_step_is_rounded_once(cuda_pkg, c, eps):
    m = 2000
    g = torch.Generator().manual_seed(c)
    x = torch.randint(-50, 51, (m, c), generator=g) * torch.randint(0, 2, (m, 1), generator=g).clamp(min=c <= 4096)
    x[:, 0] = 1
    w = torch.randn(c, generator=g).to(torch.bfloat16)
    y = rounded_norm(x, w, eps)
    want_s = (y.abs().amax(1, keepdim=True) / torch.tensor(127.0)).clamp(min=1e-30)
    xd, wd = x.to(torch.bfloat16).to(DEV), w.to(DEV)
    q, s, _ = (t.cpu() for t in cuda_pkg.ops.rmsnorm_residual_quant(xd, None, wd, eps))
    assert torch.equal(s, want_s), int((s != want_s).sum())
    assert torch.equal(q.float(), (y / want_s).round())
    if c % 32 == 0:
        code, byte = R.mx_quantize(y.double())
        q, s, _ = (t.cpu() for t in cuda_pkg.ops.rmsnorm_residual_mxfp4(xd, None, wd, eps))
        assert torch.equal(s, R.mx_tiles(byte)) and torch.equal(R.mx_codes(q) & 7, code & 7)


@pytest.mark.parametrize("c", [32, 37, 127, 128, 1001, 4096])
def test_sums_and_products_past_the_range(cuda_pkg, c):
    """A sum of squares past fp32's range is an infinity, whose row is zeros; a product past it is one, which
    the scale keeps."""
    ops = cuda_pkg.ops
    x = torch.randn((4, c), generator=torch.Generator().manual_seed(c)).to(torch.bfloat16)
    x[0], x[2] = 3e19, -3e38
    w = torch.ones(c, dtype=torch.bfloat16)
    q, s, _ = (t.cpu() for t in ops.rmsnorm_residual_quant(x.to(DEV), None, w.to(DEV)))
    assert not q[0].any() and not q[2].any() and (s[[0, 2]] == torch.tensor(1e-30)).all()
    assert torch.isfinite(s).all() and q[1].any() and q[3].any()
    x[1], x[3] = 1.0, 1.0
    x[1, 1] = 4.0                                           # the row's largest, and more than the others' mean
    w[1] = 3e38
    want = rounded_norm(x[1::2].double(), w, 1e-6)
    q, s, _ = (t.cpu() for t in ops.rmsnorm_residual_quant(x.to(DEV), None, w.to(DEV)))
    for i, row in ((1, 0), (3, 1)):
        if torch.isfinite(want[row]).all():
            assert torch.isfinite(s[i]).all() and q[i].any()
        else:
            assert torch.isinf(s[i]).all() and not q[i].any()
    assert not torch.isfinite(want[0]).all() and torch.isfinite(want[1]).all()
