"""The 8-bit layer where workspace cannot be had (tv_hip_inject_alloc_failure), each call on a fresh stream."""
import pytest
import torch

import tensorvia_amd as tv
from tests import fp8_ref as ref
from tests.test_experts_gpu import check as check_experts, make
from tests.test_fp8_gpu import DT, check_gemm

pytestmark = pytest.mark.gpu


def on_fresh_stream(fail, call):
    """call(stream) with the next `fail` requests for workspace failing."""
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    tv.lib().tv_hip_inject_alloc_failure(fail)
    try:
        out = call(stream)
    finally:
        tv.lib().tv_hip_inject_alloc_failure(0)
    stream.synchronize()
    return out


# Products that split k on workgroups of 128 columns and on tiles, and that copy their operands into padded rows for tiles (split, whole).
@pytest.mark.parametrize("fail", [1, 2, 1000])
@pytest.mark.parametrize("m,n,k,out", [(31, 300, 8323, "bf16"), (300, 1000, 8320, "f32"), (300, 1000, 8323, "f16"), (2100, 4100, 403, "bf16")])
def test_products(hip, m, n, k, out, fail):
    a, a_scale = ref.rand_rows(m, k, 31)
    w, w_scale = ref.rand_weights((n, k), 32)
    c = on_fresh_stream(fail, lambda s: tv.gemm_fp8(a, a_scale, w, w_scale, out_dtype=tv.torch_to_tv(DT[out]), stream=s))
    check_gemm(c, a, a_scale, w, w_scale, out)


@pytest.mark.parametrize("t,h,i,e,k", [(200, 256, 200, 4, 2), (200, 250, 256, 4, 2), (200, 257, 131, 4, 2)])
def test_experts_without_room_for_copies(hip, t, h, i, e, k):
    """Tiles that need W2, W1 or both in padded rows: without memory for the copy the other kernels serve the call."""
    args = make(t, h, i, e, k, 33)
    check_experts(on_fresh_stream(1, lambda s: tv.experts_fp8(*args, stream=s)), args, "bf16")
    check_experts(on_fresh_stream(0, lambda s: tv.experts_fp8(*args, stream=s)), args, "bf16")


@pytest.mark.parametrize("t,h,i,e,k", [(200, 256, 200, 4, 2), (200, 250, 256, 4, 2), (200, 256, 256, 4, 2), (40, 4096, 1376, 8, 3), (1, 512, 256, 8, 2)])
def test_experts_without_memory(hip, t, h, i, e, k):
    """Nothing at all can be allocated: an error, nothing written, and the next call is whole again."""
    args = make(t, h, i, e, k, 34)
    out = torch.full((t, h), 3.0, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(tv.TensorviaHipError) as err:
        on_fresh_stream(1000, lambda s: tv.experts_fp8(*args, out=out, stream=s))
    torch.cuda.synchronize()
    assert err.value.code == tv.TV_E_NOMEM and (out == 3).all()
    check_experts(tv.experts_fp8(*args, out=out), args, "bf16")


def test_a_capture_of_an_unprepared_stream(hip):
    """The copy of W2 cannot be had while the stream is captured: the other kernels are recorded."""
    args = make(200, 256, 200, 4, 2, 35)
    out = torch.full((200, 256), 3.0, dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()
    aligned = make(200, 256, 256, 4, 2, 36)
    with torch.cuda.stream(stream):
        tv.experts_fp8(*aligned, out=out)  # the plan's and the rows' buffers, larger than needed
        out.fill_(3.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        tv.experts_fp8(*args, out=out)
    graph.replay()
    torch.cuda.synchronize()
    check_experts(out, args, "bf16")
