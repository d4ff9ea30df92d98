"""The 8-bit layer at the limits of its index ranges."""
import pytest
import torch

import tensorvia_amd as tv
from tests import fp8_ref as ref
from tests.test_fp8_gpu import check_gemm

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
