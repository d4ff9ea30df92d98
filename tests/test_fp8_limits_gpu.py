"""The 8-bit layer at the limits of its index ranges."""
import pytest
import torch

import tensorvia_amd as tv
from tests import fp8_ref as ref
from tests.test_fp8_gpu import check_codes, check_gemm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(2100, 4100, 112), (300, 4100, 128), (2100, 4100, 256)])
def test_gemm_scales_of_distant_blocks(hip, m, n, k):
    """Blocks' scales so far apart that the k-tiles past the last one would lie beyond 2^31 bytes, on sizes that take tiles."""
    a, a_scale = ref.rand_rows(m, k, 21)
    w, w_scale = ref.rand_weights((n, k), 22)
    blocks, step = ref.up(k), 1 << 28
    far = torch.empty((blocks - 1) * step + m, device="cuda").as_strided((m, blocks), (1, step))
    far.copy_(a_scale)
    check_gemm(tv.gemm_fp8(a, far, w, w_scale), a, a_scale, w, w_scale, "bf16")


@pytest.mark.parametrize("m,k", [(1, 5), (2, 16), (16, 3)])
def test_gemm_of_more_columns_than_a_grid(hip, m, k):
    """2^27 columns and more, which the workgroups of 16 columns take in several launches: the first ones, those around the
    launches' seam and the last ones."""
    n = (1 << 27) + 1003
    a, a_scale = ref.rand_rows(m, k, 23)
    g = torch.Generator("cuda").manual_seed(24)
    w = torch.randint(0, 0x78, (n, k), dtype=torch.uint8, device="cuda", generator=g)
    w[::3] |= 0x80
    w = w.view(torch.float8_e4m3fn)
    w_scale = 0.5 + torch.rand(ref.up(n), 1, device="cuda", generator=g)
    c = tv.gemm_fp8(a, a_scale, w, w_scale)
    for first in (0, (1 << 27) - 384, n // 128 * 128 - 256):
        last = min(n, first + 700)
        check_gemm(c[:, first:last], a, a_scale, w[first:last], w_scale[first // 128:ref.up(last)], "bf16")


def test_quantize_more_blocks_than_a_grid(hip):
    """2^23 blocks of weights and one, of one column: the first ones, those around the launches' seams and the last, short one."""
    m = (1 << 30) + 57
    x = torch.zeros(m, 1, dtype=torch.bfloat16, device="cuda")
    seam = 128 << 20
    windows = [(first, min(m, first + 1024)) for first in (0, seam - 512, 7 * seam - 512, (1 << 30) - 512)]
    g = torch.Generator("cuda").manual_seed(25)
    for first, last in windows:
        x[first:last] = torch.randn(last - first, 1, device="cuda", generator=g)
    q, scale = tv.quantize_fp8(x, 128)
    for first, last in windows:
        check_codes(q[first:last], scale[first // 128:ref.up(last)], x[first:last].double(), 128, 0.0)
