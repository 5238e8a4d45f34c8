"""route_topk against a sort in 64 bits.  The choice has to be the same; a weight is rounded to float32 once (half a step,
2^-24 relative), and the float32 sum of an unbiased softmax adds at most 2 (log2 E + 4) half steps: 2^-19 in all."""
import numpy as np
import pytest
import torch

import jangq_b200 as jq
from jangq_b200 import JangqError

from oracle.mxfp4_oracle import route

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _check(logits, k, **kw):
    idx, w = jq.route_topk(logits, k, **kw)
    bias = kw.get("bias")
    ri, rw = route(logits.double().cpu().numpy(), k, kw.get("score", "softmax"),
                   None if bias is None else bias.double().cpu().numpy(), kw.get("groups", 1), kw.get("groups_kept", 1),
                   kw.get("group_top", 2), kw.get("renorm", True), kw.get("scale", 1.0))
    assert idx.dtype == torch.int32 and w.dtype == torch.float32 and tuple(idx.shape) == tuple(w.shape) == ri.shape
    assert np.array_equal(idx.cpu().numpy(), ri)
    np.testing.assert_allclose(w.double().cpu().numpy(), rw, rtol=2.0 ** -19, atol=1e-37)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,dtype,bias,groups,kept,top", [
    (1, 128, 8, "bf16", False, 1, 1, 1), (1, 1, 1, "f32", False, 1, 1, 1), (3, 7, 7, "f32", True, 1, 1, 1),
    (61, 512, 10, "f32", True, 1, 1, 2), (130, 256, 8, "f32", True, 8, 4, 2), (130, 256, 8, "bf16", False, 8, 3, 2),
    (65, 160, 6, "f16", False, 8, 3, 1), (65, 160, 6, "f16", True, 5, 2, 1), (33, 96, 40, "f32", True, 3, 2, 2),
    (17, 1024, 33, "f32", False, 32, 5, 2), (17, 1024, 1024, "bf16", True, 1, 1, 1), (9, 64, 64, "f32", False, 32, 32, 2),
    (5, 99, 11, "f32", True, 9, 1, 2), (4097, 32, 2, "bf16", False, 4, 2, 1)])
def test_route_matches_sort(score, T, E, k, dtype, bias, groups, kept, top):
    gen = torch.Generator(device="cuda").manual_seed(T * 131 + E)
    logits = (torch.randn((T, E), generator=gen, device="cuda") * 2).to(DT[dtype])
    b = torch.randn((E,), generator=gen, device="cuda") * 0.1 if bias else None
    for renorm, scale in ((True, 1.0), (False, 2.5)):
        _check(logits, k, score=score, bias=b, groups=groups, groups_kept=kept, group_top=top, renorm=renorm, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_ties_infinities_and_empty_rows(score, bias):
    """Equal logits, masked experts, rows with nothing but -inf or NaN, one +inf, scores that underflow or saturate."""
    E = 48
    rows = [np.zeros(E), np.full(E, -np.inf), np.full(E, np.nan), np.tile([1.0, 1.0, 0.5, 0.5], E // 4),
            np.where(np.arange(E) % 7 == 3, 2.0, -np.inf), np.where(np.arange(E) == 20, np.inf, 0.0),
            np.where(np.arange(E) == 11, np.nan, np.linspace(-4, 4, E)), np.linspace(-3000, 0, E), np.full(E, torch.finfo(torch.float32).min),
            np.where(np.arange(E) < 30, torch.finfo(torch.float32).min, 1.0), np.where(np.arange(E) % 2, -0.0, 0.0)]
    logits = torch.tensor(np.array(rows), dtype=torch.float32, device="cuda")
    b = torch.tensor(np.where(np.arange(E) % 5 == 0, 0.25, 0.0), dtype=torch.float32, device="cuda") if bias else None
    for groups, kept, top in ((1, 1, 1), (6, 2, 1), (6, 2, 2)):
        _check(logits, 8, score=score, bias=b, groups=groups, groups_kept=kept, group_top=top)
        _check(logits, 8, score=score, bias=b, groups=groups, groups_kept=kept, group_top=top, renorm=False)


@pytest.mark.gpu
def test_close_scores_are_told_apart():
    """Choice scores that differ by less than a float32 step: the 64-bit order decides."""
    E, T = 64, 256
    gen = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.rand((T, E), generator=gen, device="cuda") * 1e-6
    bias = torch.full((E,), 1000.0, device="cuda")                 # the float32 sum would lose every score
    _check(logits, 8, score="sigmoid", bias=bias)
    _check(logits, 8, score="softmax", bias=bias, groups=8, groups_kept=3)


@pytest.mark.gpu
def test_same_as_the_plain_router():
    gen = torch.Generator(device="cuda").manual_seed(6)
    logits = torch.randn((200, 128), generator=gen, device="cuda")
    a, b = jq.route_topk(logits, 8, scale=1.5), jq.route_softmax_topk(logits, 8, scale=1.5)
    assert torch.equal(a[0], b[0])
    torch.testing.assert_close(a[1], b[1], rtol=1e-5, atol=0)


@pytest.mark.gpu
def test_views_streams_and_graphs():
    gen = torch.Generator(device="cuda").manual_seed(7)
    big = torch.randn((40, 300), generator=gen, device="cuda")
    _check(big[:, 7:135], 4, score="sigmoid")                      # rows with a pitch, unaligned
    _check(big.t()[:96, :32], 4)                                   # columns
    _check(big[3:4].expand(5, 300)[:, :256], 4)                    # broadcast rows
    assert jq.route_topk(big[:0], 4)[0].shape == (0, 4)
    bias = torch.randn((300,), generator=gen, device="cuda", dtype=torch.float64)[::1]
    _check(big, 5, bias=bias.float())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = jq.route_topk(big, 8, groups=10, groups_kept=4)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = jq.route_topk(big, 8, groups=10, groups_kept=4)
        first = big.clone()
        big.copy_(torch.randn((40, 300), generator=gen, device="cuda"))
        graph.replay()
        other = [g.clone() for g in got]
        big.copy_(first)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not torch.equal(other[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(k=0), dict(k=65), dict(k=9, groups=8, groups_kept=1), dict(k=2, groups=5), dict(k=2, groups=0),
                                dict(k=2, groups=64), dict(k=2, groups=8, groups_kept=9), dict(k=2, groups=8, groups_kept=0),
                                dict(k=2, groups=8, groups_kept=2, group_top=3), dict(k=2, groups=8, groups_kept=2, group_top=0),
                                dict(k=2, score="relu"), dict(k=-1), dict(k=1 << 40), dict(k=(1 << 32) + 2)])
def test_refusals(kw):
    logits = torch.zeros((3, 64), device="cuda")
    with pytest.raises(JangqError):
        jq.route_topk(logits, **kw)


@pytest.mark.gpu
def test_refused_tensors():
    with pytest.raises(JangqError):
        jq.route_topk(torch.zeros((2, 1025), device="cuda"), 2)
    with pytest.raises(JangqError):
        jq.route_topk(torch.zeros((64,), device="cuda"), 2)
    with pytest.raises(JangqError):
        jq.route_topk(torch.zeros((2, 64), dtype=torch.float64, device="cuda"), 2)
    with pytest.raises(JangqError):
        jq.route_topk(torch.zeros((2, 64), device="cuda"), 2, bias=torch.zeros(63, device="cuda"))
    with pytest.raises(JangqError):
        jq.route_topk(torch.zeros((2, 64), device="cuda"), 2, bias=torch.zeros(64))


def test_cpu_logits_are_refused():
    with pytest.raises(JangqError):
        jq.route_topk(torch.zeros((2, 64)), 2)
