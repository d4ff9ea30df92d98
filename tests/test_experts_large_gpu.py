"""Layers of experts with 8192 slots and more, whose tiles do without exact sums for bf16 results."""
import pytest
import torch

import tensorvia_amd as tv
from tests.test_experts_gpu import check, make
from tests.test_fp8_paths_gpu import framed

pytestmark = pytest.mark.gpu


# Tiles of 256 rows (whole and short blocks, operands of either product in padded rows, k past 64 blocks in either) and of 128 (many
# experts); all rows with one expert.
@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("t,h,i,e,k", [(4200, 256, 256, 8, 2), (2800, 304, 208, 5, 3), (4200, 250, 131, 8, 2), (4200, 256, 200, 8, 2), (4200, 257, 256, 8, 2),
                                       (4200, 8320, 128, 2, 2), (4200, 128, 8320, 2, 2), (4200, 256, 200, 200, 2), (8200, 384, 144, 1, 1)])
def test_large_layers(hip, t, h, i, e, k, out):
    args = make(t, h, i, e, k, t + h + i)
    args[7][t // 2:t // 2 + 3] = -1
    args[7][5, 0] = e
    c, intact = framed(t, h, out)
    tv.experts_fp8(*args, out=c)
    check(c, args, out)
    assert intact()


def test_streams_and_graphs(hip):
    """The same bits on every run, on two streams at once, and in replays."""
    args = make(4200, 256, 256, 8, 2, 41)
    want = tv.experts_fp8(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(want) for _ in streams]
    for _ in range(3):
        for s, o in zip(streams, outs):
            tv.experts_fp8(*args, out=o, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        tv.experts_fp8(*args, out=outs[0])
    for _ in range(3):
        outs[0].zero_()
        tv.experts_fp8(*args, out=outs[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_nan_stays_with_its_token(hip):
    args = make(4200, 256, 128, 4, 2, 42)
    args[0].view(torch.uint8)[1, 77] = 0x7F
    got = tv.experts_fp8(*args)
    assert torch.isnan(got[1]).all() and int(torch.isnan(got).sum()) == 256
