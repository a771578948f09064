"""SwiGLU + MXFP4 where the gate's silu leaves fp32's range and its product with `up` does not."""
import operator_refs as R
import pytest
import torch
from test_gpu_mxfp4 import near_border

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("m,k", [(1, 32), (130, 96), (257, 1024)])
@pytest.mark.parametrize("largest", [0.0, 30.0, 126.0])
def test_far_gates(cuda_pkg, m, k, largest):
    """Gates from -60 to -200, up to 2^largest (0: of the size that makes the product normal)."""
    g = torch.Generator().manual_seed(m + k)
    gate = -60 - 140 * torch.rand((m, k), generator=g)
    if largest:
        up = torch.exp2(largest * torch.rand((m, k), generator=g)) * torch.where(torch.rand((m, k), generator=g) < 0.5, -1.0, 1.0)
    else:
        gate.clamp_(min=-170)
        up = torch.exp2((-gate * 1.4427 - 120).clamp(max=126)) * torch.randn((m, k), generator=g).clamp(-1.9, 1.9)
    gate[:, 5] = 3.0                                        # a near gate among far ones
    up[:, 5] = 2.0 ** -100
    x = torch.cat((gate, up), 1).to(torch.bfloat16)
    gd, ud = x[:, :k].double(), x[:, k:].double()
    want = gd * torch.sigmoid(gd) * ud
    q, s = cuda_pkg.ops.swiglu_quantize_mxfp4(x.to(DEV))
    # the fast exponential (gates down to -80) is within 2 + 1.173 |g| units of 2^-23 (96), the far one four
    # times two; reciprocal, sum and products one each, five at most; a subnormal result (all
    # elements below 2^-129 round to zero) half of 2^-149 more per product, 5 * 2^-21 of it: 101 * 2^-23 + 3e-6
    near_border(want, R.mx_bytes(s.cpu(), m, k), R.mx_codes(q.cpu()), 1.6e-5)
    if largest == 126.0:
        assert (want[gd < -88].abs() > 2.0 ** -126).any()   # the range is reached


def test_infinite_and_nan_gates(cuda_pkg):
    x = torch.randn((4, 128), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    x[0, 3], x[1, 40] = float("-inf"), float("nan")         # -inf * 0 is a NaN in the formula
    x[2, 7], x[2, 71] = -3e38, 3e38                         # e^g is 0: the product is -0
    q, s = cuda_pkg.ops.swiglu_quantize_mxfp4(x.to(DEV))
    byte = R.mx_bytes(s.cpu(), 4, 64)
    assert byte[0, 0] == 255 and byte[1, 1] == 255
    assert (byte[0, 1] < 255) and (byte[1, 0] < 255) and (byte[2:] < 255).all() and R.mx_codes(q.cpu())[2, 7] & 7 == 0
