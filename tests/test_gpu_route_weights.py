"""Weights of route_topk where nothing cancels in them: each is the 64-bit score rounded to float32 once."""
import numpy as np
import pytest
import torch

import jangq_b200 as jq

from oracle.mxfp4_oracle import route

HALF_STEP = 2.0 ** -24 * (1 + 2.0 ** -20)                  # of float32, and what 64-bit exponentials and sums may add


def _check(logits, k, bias=None, **kw):
    idx, w = jq.route_topk(logits, k, bias=bias, **kw)
    ri, rw = route(logits.double().cpu().numpy(), k, kw.get("score", "softmax"), None if bias is None else bias.double().cpu().numpy(),
                   kw.get("groups", 1), kw.get("groups_kept", 1), kw.get("group_top", 2), kw.get("renorm", True), kw.get("scale", 1.0))
    assert np.array_equal(idx.cpu().numpy(), ri)
    np.testing.assert_allclose(w.double().cpu().numpy(), rw, rtol=HALF_STEP, atol=2.0 ** -150)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,groups,kept", [(1, 128, 8, 1, 1), (300, 33, 5, 1, 1), (200, 256, 8, 8, 4), (100, 512, 10, 1, 1), (50, 1024, 32, 1, 1)])
def test_softmax_weights_without_renormalisation(T, E, k, groups, kept, dtype):
    gen = torch.Generator(device="cuda").manual_seed(E + T)
    logits = (torch.randn((T, E), generator=gen, device="cuda") * 2).to(dtype)
    _check(logits, k, groups=groups, groups_kept=kept, group_top=1, renorm=False)
    bias = torch.randn((E,), generator=gen, device="cuda") * 0.1
    _check(logits, k, bias, groups=groups, groups_kept=kept, renorm=False)


@pytest.mark.gpu
def test_renormalised_weights_of_experts_with_next_to_no_score():
    """A bias that takes experts whose scores add up to the size of the 1e-20 beside their sum: the sum no longer cancels."""
    T, E, k = 64, 96, 4
    gen = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn((T, E), generator=gen, device="cuda")
    logits[:, :32] += torch.linspace(30.0, 60.0, T, device="cuda")[:, None]
    bias = torch.where(torch.arange(E, device="cuda") < 32, 0.0, torch.linspace(7.0, 9.0, E, device="cuda"))
    _check(logits, k, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k,groups,kept", [(33, 1, 1), (64, 4, 2), (96, 1, 1)])
def test_many_experts_with_next_to_no_score(score, k, groups, kept):
    """More than 32 experts: no score is rounded before the sum of all of them is known, below float32's range neither."""
    T, E = 40, 128
    gen = torch.Generator(device="cuda").manual_seed(k)
    logits = torch.randn((T, E), generator=gen, device="cuda") - torch.linspace(0.0, 120.0, T, device="cuda")[:, None]
    logits[:, :32] += torch.linspace(0.0, 150.0, T, device="cuda")[:, None]
    bias = torch.where(torch.arange(E, device="cuda") < 32, 0.0, torch.linspace(7.0, 9.0, E, device="cuda"))
    for renorm in (True, False):
        _check(logits, k, bias, score=score, groups=groups, groups_kept=kept, renorm=renorm)
        _check(logits, k, None, score=score, groups=groups, groups_kept=kept, group_top=1, renorm=renorm)
