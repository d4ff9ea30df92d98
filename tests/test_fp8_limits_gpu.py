"""The 8-bit layer at the limits of its index ranges."""
import pytest
import torch

import tensorvia_amd as tv
from tests import fp8_ref as ref
from tests.test_experts_gpu import check as check_experts
from tests.test_fp8_gpu import DT, check_codes, check_gemm

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


def shared_experts(t, h, i, e, k, seed):
    """Arguments of a layer whose experts share one pair of codes (strides of 0) under scales of their own."""
    g = torch.Generator("cuda").manual_seed(seed)
    a, a_scale = ref.rand_rows(t, h, seed)
    w1, w2 = (ref.rand_weights(shape, seed + 1)[0].expand(e, *shape[1:]) for shape in ((1, 2, i, h), (1, h, i)))
    w1_scale = (0.02 / 107) * torch.exp(0.2 * torch.randn(e, 2, ref.up(i), ref.up(h), device="cuda", generator=g))
    w2_scale = (0.02 / 107) * torch.exp(0.2 * torch.randn(e, ref.up(h), ref.up(i), device="cuda", generator=g))
    weights, ids = torch.softmax(torch.randn(t, e, device="cuda", generator=g), -1).topk(k, -1)
    return [a, a_scale, w1, w1_scale, w2, w2_scale, (weights / weights.sum(-1, keepdim=True)).contiguous(), ids.to(torch.int32)]


def check_tokens(got, args, tokens, out):
    tokens = torch.tensor(tokens, device="cuda")
    part = [x.view(torch.uint8)[tokens].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[tokens].contiguous() for x in args[:2]]
    check_experts(got[tokens], part + args[2:6] + [args[6][tokens], args[7][tokens]], out)


@pytest.mark.parametrize("t,i,e,k,out", [(2816, 448_000, 1024, 8, "bf16"), (1024, 1_000_000, 1024, 1, "f32")])
def test_experts_of_more_workgroups_than_a_grid(hip, t, i, e, k, out):
    """Widths at which the tiles' grid, and that of the workgroups of 128 columns, would hold too many threads."""
    args = shared_experts(t, 16, i, e, k, 26)
    check_tokens(tv.experts_fp8(*args, out_dtype=tv.torch_to_tv(DT[out])), args, [0, t // 2, t - 1], out)


def test_one_token_of_more_columns_than_a_grid(hip):
    """A row of 2^26 elements and more through one expert.  Its first 1024 elements are not zero; the results' first, middle and
    last ones."""
    h, i, part = (1 << 26) + 2048, 16, 1024
    g = torch.Generator("cuda").manual_seed(27)

    def codes(*shape):
        w = torch.randint(0, 0x70, shape, dtype=torch.uint8, device="cuda", generator=g)
        w[..., ::3] |= 0x80
        return w.view(torch.float8_e4m3fn)
    a = torch.zeros(1, h, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    a[:, :part] = codes(1, part)
    w1, w2 = codes(1, 2, i, h), codes(1, h, i)
    scales = [1e-3 + 1e-3 * torch.rand(shape, device="cuda", generator=g) for shape in ((1, ref.up(h)), (1, 2, 1, ref.up(h)), (1, ref.up(h), 1))]
    weights, ids = torch.full((1, 1), 0.5, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    got = tv.experts_fp8(a, scales[0], w1, scales[1], w2, scales[2], weights, ids)
    for first in (0, 1 << 25, h - part):
        block = slice(first // 128, (first + part) // 128)
        check_experts(got[:, first:first + part], [a[:, :part], scales[0][:, :8], w1[..., :part], scales[1][..., :8], w2[:, first:first + part],
                                                   scales[2][:, block], weights, ids], "bf16")
