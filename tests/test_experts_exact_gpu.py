"""The layer of experts on values that fp32 holds exactly at every step: fp32 results are the sums themselves."""
import pytest
import torch

import tensorvia_amd as tv
from tests import fp8_ref as ref

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def make(t, h, i, e, k, seed):
    """gate = 32, whose sigmoid is 1 in fp32, and up = integers of -14 to 14, 14 in every block of 128: the inner rows are 32 * up with
    scale 1, and those are codes.  W2 holds values of 2^-9 to 7 * 2^-9 and two of 448 in each row, so a block's products
    span 22 bits; all sums are multiples of 2^-4 below 2^20, 24 bits."""
    g = torch.Generator().manual_seed(seed)
    column = 1 + torch.randint(h - 1, (t,), generator=g)
    a = torch.zeros(t, h)
    a[:, 0] = 32.0
    a[torch.arange(t), column] = 1.0
    w1 = torch.zeros(e, 2, i, h)
    w1[:, 0, :, 0] = 1.0
    w1[:, 1, :, 1:] = torch.randint(-14, 15, (e, i, h - 1), generator=g).float()
    w1[:, 1, ::128, 1:] = 14.0
    w2 = torch.randint(-7, 8, (e, h, i), generator=g).float() * 2.0 ** -9
    for _ in range(2):
        at = torch.randint(i, (e, h, 1), generator=g)
        w2.scatter_(2, at, 448.0 * (1 - 2 * torch.randint(2, (e, h, 1), generator=g).float()))
    ids = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(t)]).to(torch.int32)
    one = lambda *shape: torch.ones(*shape, device="cuda")  # noqa: E731
    args = [a.to(F8).cuda(), one(t, ref.up(h)), w1.to(F8).cuda(), one(e, 2, ref.up(i), ref.up(h)), w2.to(F8).cuda(),
            one(e, ref.up(h), ref.up(i)), one(t, k), ids.cuda()]
    want = torch.zeros(t, h, dtype=torch.float64)
    for x in range(e):
        token = (ids == x).any(1).nonzero().flatten()
        want[token] += (32 * w1[x, 1].double()[:, column[token]]).t() @ w2[x].double().t()
    return args, want


# One and few tokens without a plan; workgroups of 16 columns; of 128 columns and 16, 32 and 64 rows; k in parts; rows that are not aligned.
@pytest.mark.parametrize("t,h,i,e,k", [(1, 512, 640, 4, 2), (1, 257, 131, 4, 2), (3, 300, 208, 16, 2), (17, 300, 129, 5, 2), (40, 256, 256, 8, 2), (5, 64, 2600, 3, 2),
                                       (26, 256, 640, 64, 2), (300, 256, 256, 64, 2), (900, 256, 256, 64, 2), (300, 251, 263, 64, 2),
                                       (60, 128, 8320, 2, 1), (1200, 128, 256, 4, 2)])
def test_fp32_results_are_exact(hip, t, h, i, e, k):
    args, want = make(t, h, i, e, k, t + h + i)
    got = tv.experts_fp8(*args, out_dtype=tv.FLOAT32)
    assert (want.abs() < 2.0 ** 20).all() and (want * 16 == (want * 16).round()).all()
    off = (got.double().cpu() - want).abs()
    assert torch.equal(got.double().cpu(), want), f"{int((off > 0).sum())} of {off.numel()} off, by up to {float(off.max())}"


@pytest.mark.parametrize("t,h,i,e,k", [(60, 1536, 512, 8, 4), (50, 512, 384, 8, 4), (250, 1536, 512, 8, 4)])
def test_bf16_results_of_few_slots(hip, t, h, i, e, k):
    """The error's norm against 64 bits, call by call: the rounding to bf16, at most 2^-8 / sqrt(3) of the result (half an ulp of
    the smallest mantissa, evenly spread), and 2^-10 for the codes that exact sums still move and the second product.  Where the first
    product's sums are cut, a few moved codes of large values make some of the calls several times worse."""
    from tests.test_experts_gpu import make as layer
    for seed in range(40):
        args = layer(t, h, i, e, k, 1000 + seed)
        want, _ = ref.experts(*args)
        got = tv.experts_fp8(*args).double()
        error = float((got - want).norm() / want.norm())
        assert error <= 2.0 ** -8 / 3 ** 0.5 + 2.0 ** -10, (seed, error)
