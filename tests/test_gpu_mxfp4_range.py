"""MXFP4 mat-vec with activations and scales from end to end of their types.

A product of the mat-vec is rounded once to its output type; the sums are float32, at most 16 products per step, each step off
by at most a float32 step of the magnitudes summed so far; a bf16 activation is off by at most 2^-39 of the largest of its block
of 32 (f16 pairs at 2^14 to 2^15 of that block, half of their smallest step 2^-24):
|error| <= eps/2 |y| + (K/16 + 32) 2^-23 sum |x w| + 2^-39 sum_blocks max |x| sum |w|."""
import numpy as np
import pytest
import torch

import jangq_b200 as jq

from oracle import mxfp4_oracle as mo


def _bank(rng, shape, byte):
    """Random codes [.., N, K] with the scale bytes [.., N, K/32]: (codes, scales) on the GPU and their float64 values."""
    code = rng.integers(0, 16, shape).astype(np.uint8)
    words, byte = mo.pack(code), byte.astype(np.uint8)
    return torch.from_numpy(words.view(np.int32)).cuda(), torch.from_numpy(byte).cuda(), mo.values(words, byte)


def _bf16(values):
    return torch.from_numpy(np.asarray(values, np.float64)).to(torch.bfloat16).cuda()


def _check(y, x, w):
    """y [M, N] against x [M, K] . w [N, K]^T; the references stay far below the largest float32"""
    K = x.shape[1]
    ref, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    largest = np.abs(x).reshape(len(x), -1, 32).max(-1)
    rounded = largest @ np.abs(w).reshape(len(w), -1, 32).sum(-1).T
    tol = 2.0 ** -8 * np.abs(ref) + (K / 16 + 32) * 2.0 ** -23 * mag + 2.0 ** -39 * rounded
    err = np.abs(y.double().cpu().numpy() - ref)
    assert np.isfinite(ref).all() and np.all(err <= tol), float((err / np.maximum(tol, 1e-300)).max())


def _ends(rng, M, N, K):
    """Activations whose blocks lie anywhere between 2^-133 and 2^127, and scale bytes that bring each block's share of every
    result to between 2^-8 and 2^16."""
    p = rng.integers(-130, 128, K // 32)
    p[:4] = (127, -126, 113, -100)[:len(p[:4])]
    x = rng.uniform(1.0, 1.99, (M, K)) * rng.choice([-1.0, 1.0], (M, K)) * np.exp2(np.repeat(p, 32).astype(np.float64))
    x = _bf16(np.where(rng.random((M, K)) < 0.1, 0.0, x))
    byte = np.clip(127 - p[None] + rng.integers(-2, 3, (N, K // 32)), 0, 254)
    return x, byte


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 40, 128), (1, 33, 4128), (2, 40, 2048), (3, 40, 128), (5, 17, 800), (8, 130, 2048), (20, 40, 288)])
def test_every_size_of_activation_against_scales_of_the_other_end(M, N, K):
    rng = np.random.default_rng(M * K)
    x, byte = _ends(rng, M, N, K)
    wq, s, w = _bank(rng, (N, K), byte)
    _check(jq.mxfp4_matmul(x, wq, s), x.double().cpu().numpy(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("p", [127, 126, 122, 114, 113, 100, -86, -87, -100, -120, -126, -130, -133])
@pytest.mark.parametrize("M", [1, 5])
def test_one_large_or_small_activation(M, p):
    """A power of two alone in its row and block: every product is exact."""
    N, K = 24, 96
    rng = np.random.default_rng(p + 200)
    byte = np.full((N, K // 32), min(max(127 - p, 0), 254))
    wq, s, w = _bank(rng, (N, K), byte)
    x = np.zeros((M, K))
    at = (np.arange(M) * 29 + 7) % K
    x[np.arange(M), at] = 2.0 ** p
    y = jq.mxfp4_matmul(_bf16(x), wq, s)
    assert np.array_equal(y.double().cpu().numpy(), (2.0 ** p) * w[:, at].T)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 4])
def test_products_beyond_the_type_and_zeros_beside_them(M):
    """A product above the largest number is infinite, one below the smallest zero, and neither makes a NaN of a zero code or a
    zero activation in its block."""
    N, K = 16, 64
    code = np.zeros((N, K), np.uint8)
    code[1:, 3] = 2                                        # weight 1 at column 3, row 0 has none
    words = mo.pack(code)
    wq = torch.from_numpy(words.view(np.int32)).cuda()
    for p, byte, want in ((127, 254, np.inf), (126, 150, np.inf), (-126, 1, 0.0), (-133, 0, 0.0), (127, 0, 1.0), (-126, 253, 1.0)):
        s = torch.full((N, K // 32), byte, dtype=torch.uint8, device="cuda")
        x = np.zeros((M, K))
        x[:, 3], x[:, 10] = 2.0 ** p, -(2.0 ** p)          # column 10 meets zero codes only
        y = jq.mxfp4_matmul(_bf16(x), wq, s).double().cpu().numpy()
        assert not y[:, 0].any() and np.array_equal(y[:, 1:], np.full((M, N - 1), want)), (p, byte)


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,N,K", [(1, 8, 16, 40, 128), (7, 3, 5, 33, 96), (60, 1, 4, 20, 2080)])
def test_routed_pairs(T, k, E, N, K):
    """The mat-vec per pair; rows of several tokens follow one another in a CTA, ordinary ones among those of extreme size."""
    rng = np.random.default_rng(T + K)
    x, byte = _ends(rng, T, E * N, K)
    wq, s, w = _bank(rng, (E, N, K), byte.reshape(E, N, -1))
    idx = rng.integers(0, E, (T, k))
    y = jq.mxfp4_gather_matmul(x, wq, s, rhs_indices=torch.from_numpy(idx).int().cuda()).reshape(T, k, N)
    xn = x.double().cpu().numpy()
    for t in range(T):
        for j in range(k):
            _check(y[t, j][None], xn[t:t + 1], w[idx[t, j]])
    # every other token is a row of ordinary activations
    x2 = x.clone()
    x2[::2] = _bf16(rng.standard_normal((len(x[::2]), K)))
    wq, s, w = _bank(rng, (E, N, K), rng.integers(118, 124, (E, N, K // 32)))
    y = jq.mxfp4_gather_matmul(x2, wq, s, rhs_indices=torch.from_numpy(idx).int().cuda()).reshape(T, k, N)
    xn = x2.double().cpu().numpy()
    for t in range(0, T, 2):
        for j in range(k):
            _check(y[t, j][None], xn[t:t + 1], w[idx[t, j]])
