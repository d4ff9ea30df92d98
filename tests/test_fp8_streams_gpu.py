"""Results that a call allocates while it runs on another stream than the current one."""
import pytest
import torch

import tensorvia_amd as tv
from tests import fp8_ref as ref

pytestmark = pytest.mark.gpu

M, N, K = 500, 640, 384


@pytest.fixture(scope="module")
def inputs(hip):
    g = torch.Generator().manual_seed(1)
    x = [torch.randn(M, K, generator=g).bfloat16().cuda() for _ in range(2)]
    b = torch.randn(K, N, generator=g).bfloat16().cuda()
    w, w_scale = ref.rand_weights((N, K), 2)
    quantised = [tv.quantize_fp8(y) for y in x]
    w1, w1_scale = ref.rand_weights((4, 2, 256, K), 3)
    w2, w2_scale = ref.rand_weights((4, K, 256), 4)
    weights, ids = tv.route(torch.randn(M, 4, generator=g).cuda(), 2)
    gamma = torch.ones(K, device="cuda").bfloat16()
    calls = {
        "gemm": lambda i, s: [tv.gemm(x[i], b, stream=s)],
        "quantize": lambda i, s: list(tv.quantize_fp8(x[i], stream=s)),
        "quantize_weights": lambda i, s: list(tv.quantize_fp8(x[i], 128, stream=s)),
        "norm": lambda i, s: list(tv.rms_norm_fp8(x[i], gamma, x[1], normed=True, stream=s)),
        "gemm_fp8": lambda i, s: [tv.gemm_fp8(*quantised[i], w, w_scale, stream=s)],
        "route": lambda i, s: list(tv.route(x[i], 8, stream=s)),
        "experts": lambda i, s: [tv.experts_fp8(*quantised[i], w1, w1_scale, w2, w2_scale, weights, ids, stream=s)],
    }
    for call in calls.values():
        call(0, None)
    torch.cuda.synchronize()
    return calls


def same(got, want):
    return all(torch.equal(g.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8)) for g, w in zip(got, want))


def delay():
    torch.cuda._sleep(20_000_000)


CALLS = ["gemm", "quantize", "quantize_weights", "norm", "gemm_fp8", "route", "experts"]


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_results_are_not_memory_that_queued_work_still_writes(inputs, name, handle):
    """Tensors of the results' sizes, freed while the current stream has yet to fill them."""
    call = inputs[name]
    want = call(0, None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    delay()
    old = [torch.empty_like(t) for t in want for _ in range(2)]
    for t in old:
        t.view(torch.uint8).fill_(7) if t.is_contiguous() else t.t().view(torch.uint8).fill_(7)
    del old, t
    got = call(0, side.cuda_stream if handle else side)
    torch.cuda.synchronize()
    assert same(got, want)


@pytest.mark.parametrize("name", CALLS)
def test_results_that_queued_work_still_reads_are_not_overwritten(inputs, name):
    """The current stream waits for the call, reads its results behind other work, and they are freed before it does: a second
    call on the same stream gets other memory."""
    call = inputs[name]
    want = call(0, None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = call(0, side)
    torch.cuda.current_stream().wait_stream(side)
    delay()
    copies = [t.clone() for t in got]
    del got
    call(1, side)
    torch.cuda.synchronize()
    assert same(copies, want)


def test_the_null_stream_s_handle(inputs):
    """0 is the default stream, also while another one is current."""
    want = inputs["gemm_fp8"](0, None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = inputs["gemm_fp8"](0, 0)
    torch.cuda.synchronize()
    assert same(got, want)
