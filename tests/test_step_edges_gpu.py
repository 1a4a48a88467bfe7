"""Edges of the serving-step operators (squish_b200.ops.step) on the GPU: each test is a call that the
documentation allows, or a refusal, next to the limits of an operator."""
import numpy as np
import pytest
import torch

from squish_b200 import ops

from ._step_refs import route_ref

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- routing
def opposite_biases(B, score, groups, gsize, T, seed):
    """Logits and a bias with which every group's two best choice values are near +B and -B and the
    groups' exact sums lie a few fp32 rounding steps of B apart (rows with an exact tie are dropped)."""
    g = torch.Generator().manual_seed(seed)
    E = groups * gsize
    s1 = 0.05 + 0.6 * torch.rand(T, groups, generator=g, dtype=torch.float64)
    total = 0.765 + (2 * torch.rand(T, groups, generator=g, dtype=torch.float64) - 1) * B * 2.0**-22
    s = torch.full((T, groups, gsize), 0.01, dtype=torch.float64)
    s[..., 0], s[..., 1] = s1, total - s1
    s = s.view(T, E)
    x = torch.log(s / (1 - s)) if score == "sigmoid" else torch.log(s)
    bias = torch.full((groups, gsize), -2.0 * B)
    bias[:, 0], bias[:, 1] = B, -B
    x, bias = x.float(), bias.view(E).float()
    exact = torch.sigmoid(x.double()) if score == "sigmoid" else torch.softmax(x.double(), -1)
    sums = (exact + bias.double()).view(T, groups, gsize)[..., :2].sum(-1).sort(-1).values
    keep = (sums[:, 1:] - sums[:, :-1]).amin(-1) > B * 2.0**-44  # (64-bit sums resolve 2^-52 B)
    return x[keep], bias


@pytest.mark.parametrize("B", [16.0, 100.0, 1e4])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups,gsize", [(8, 8), (6, 11), (4, 2)])
def test_group_sums_of_opposite_biases_are_ranked_exactly(cuda, B, score, groups, gsize):
    x, bias = opposite_biases(B, score, groups, gsize, 2000, int(B) + groups)
    assert x.shape[0] > 1500
    T, k = x.shape[0], groups // 2
    ids = torch.empty(T * k, dtype=torch.int32, device=cuda)
    w = torch.empty(T * k, device=cuda)
    kw = dict(score=score, groups=groups, top_groups=groups // 2, group_score="top2")
    ops.moe_route_scored(x.to(cuda), k, ids, w, bias=bias.to(cuda), **kw)
    want, _ = route_ref(x, k, bias=bias, **kw)
    assert np.array_equal(ids.view(T, k).cpu().numpy(), want)
