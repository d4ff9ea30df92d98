"""Routing of long batches, which 16 lanes a token serve, against short ones of the same rows, which a wave a token serves, bit for
bit; and the short ones against the definition in 64 bits."""
import pytest
import torch

import tensorvia_amd as tv
from tests.test_route_gpu import DT, INF, check

pytestmark = pytest.mark.gpu

T = 4099  # from 4096 tokens on


def rows(e, dt, seed):
    """Logits with ties (16-bit types have many), experts masked by -inf, NaN and the type's lowest value, rows with fewer than k
    experts and with none."""
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(T, e, generator=g)
    x[torch.rand(T, e, generator=g) < 0.02] = -INF
    x[torch.rand(T, e, generator=g) < 0.01] = float("nan")
    x[torch.rand(T, e, generator=g) < 0.005] = INF
    x[5::97] = 1.0
    x[6::97, 1:] = -INF
    x[7::97] = -INF
    x[8::97] = float("nan")
    x[9::97, e // 2:] = torch.finfo(DT[dt]).min
    x[10::97] = torch.finfo(DT[dt]).min
    return x.to(DT[dt]).cuda()


def compare(logits, k, **kw):
    weights, ids = tv.route(logits, k, **kw)
    for lo in range(0, T, 2050):
        w, i = tv.route(logits[lo:lo + 2050], k, **kw)
        assert torch.equal(ids[lo:lo + 2050], i), int((ids[lo:lo + 2050] != i).any(1).sum())
        assert torch.equal(weights[lo:lo + 2050], w)
    for lo in (0, T - 110):
        check(logits[lo:lo + 110], k, **kw)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,k", [(1, 1), (3, 2), (8, 8), (16, 4), (17, 16), (60, 8), (64, 8), (65, 5), (128, 16), (160, 6), (255, 9), (256, 8)])
def test_choice(hip, e, k, scoring, dt):
    logits = rows(e, dt, e + k)
    bias = 0.1 * torch.randn(e, generator=torch.Generator().manual_seed(e))
    bias[1::7] = -INF
    bias[2::9] = float("nan")
    compare(logits, k, scoring=scoring)
    compare(logits, k, scoring=scoring, bias=bias.cuda(), renormalize=False, scale=2.5)


@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups,topk_groups,k", [(12, 3, 2, 4), (16, 16, 5, 5), (15, 5, 3, 8), (60, 3, 1, 16), (60, 5, 2, 6), (60, 6, 4, 8), (60, 12, 5, 7), (60, 15, 9, 12),
                                                    (64, 8, 3, 8), (64, 2, 1, 8), (65, 13, 4, 6), (128, 16, 7, 10), (160, 10, 3, 8), (256, 4, 2, 8), (256, 8, 4, 8)])
def test_groups(hip, e, groups, topk_groups, k, scoring, group_top):
    logits = rows(e, "f32", e + groups)
    bias = (0.3 * torch.randn(e, generator=torch.Generator().manual_seed(e))).cuda()
    bias[e // 3] = -INF
    compare(logits, k, scoring=scoring, bias=bias, groups=groups, topk_groups=topk_groups, group_top=group_top)
    compare(logits.bfloat16(), k, scoring=scoring, groups=groups, topk_groups=topk_groups, group_top=group_top)


@pytest.mark.parametrize("e", [7, 60, 100, 200])
def test_strided_rows(hip, e):
    """Rows between other elements that are not numbers."""
    buf = torch.full((T, e + 13), float("nan"), device="cuda").bfloat16()
    logits = buf[:, 5:5 + e]
    logits.copy_(rows(e, "bf16", e))
    want = tv.route(logits.contiguous(), min(e, 8))
    got = tv.route(logits, min(e, 8))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
