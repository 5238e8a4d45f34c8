"""The product of two MXFP4 operands at sizes that reach every form and tile width that the rule chooses (which size reaches which
is checked by test_mxfp4_form_emulation.py).

A product is rounded once to its type on top of float32 sums of exact products:
|error| <= eps/2 |y| + (K/16 + 32) 2^-23 sum |x w|."""
import pytest
import torch

import jangq_b200 as jq


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(262, 11008, 32), (289, 11008, 64), (343, 11008, 96), (136, 11008, 288), (150, 11008, 544),
                                   (180, 11008, 64), (240, 11008, 1056), (500, 11008, 288), (512, 14336, 288), (1, 20000, 4128),
                                   (60, 11008, 4128), (128, 14400, 2080), (33, 2000, 2080), (300, 130, 5152), (70, 300, 4128),
                                   (16, 4000, 8224), (262, 11001, 32), (343, 11001, 96), (240, 11001, 288)])
def test_every_form(M, N, K, out):
    gen = torch.Generator(device="cuda").manual_seed(M + N + K)
    wq, s = jq.mxfp4_quantize(torch.randn((N, K), generator=gen, device="cuda") * 0.02)
    xq, xs = jq.mxfp4_quantize(torch.randn((M, K), generator=gen, device="cuda"))
    w, x = (jq.mxfp4_dequantize(*q, torch.float32).double() for q in ((wq, s), (xq, xs)))
    y = jq.mxfp4_matmul(xq, wq, s, x_scales=xs, dtype=out)
    ref, mag = x @ w.t(), x.abs() @ w.abs().t()
    assert y.dtype == out and y.shape == ref.shape
    assert bool(((y.double() - ref).abs() <= torch.finfo(out).eps / 2 * ref.abs() + (K / 16 + 32) * 2.0 ** -23 * mag).all())
    jq._lib.check(jq._lib.load().jq_device_status())
