"""MXFP4 quantizer, products and experts' products against plain 64-bit numpy.

Codes, scales and dequantized numbers are exact.  A product is rounded once to its output type (half a step of the value)
on top of float32 sums; the tensor cores add at least 16 products per step, each step off by at most a float32 step of the
magnitudes summed so far: |error| <= eps/2 |y| + (K/16 + 32) 2^-23 sum |x w|  (32: sums across warps, CTAs and blocks)."""
import numpy as np
import pytest
import torch

import jangq_b200 as jq
from jangq_b200 import JangqError, moe

from oracle import mxfp4_oracle as mo

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _rand(seed, shape, dtype="f32", scale=1.0):
    g = np.random.default_rng(seed)
    return torch.tensor(g.standard_normal(shape) * scale, dtype=torch.float32).to(DT[dtype]).cuda()


def _np(t):
    return t.double().cpu().numpy()


def _packed(seed, shape, scale=0.02):
    """Random MXFP4 weights: (codes int32, scales uint8) on the GPU and their float64 values."""
    w = np.random.default_rng(seed).standard_normal(shape) * scale
    code, byte = mo.quantize(w.reshape(-1, shape[-1]))
    words, byte = mo.pack(code).reshape(shape[:-1] + (-1,)), byte.reshape(shape[:-1] + (-1,))
    return torch.from_numpy(words.view(np.int32)).cuda(), torch.from_numpy(byte).cuda(), mo.values(words, byte)


def _close(y, x, w, K):
    """y [M, N] against x [M, K] . w [N, K]^T in 64 bits"""
    ref, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    step = torch.finfo(y.dtype).eps / 2
    tol = step * np.abs(ref) + (K / 16 + 32) * 2.0 ** -23 * mag + torch.finfo(y.dtype).tiny
    err = np.abs(_np(y) - ref)
    assert y.shape == ref.shape and np.all(err <= tol), float((err / tol).max())


# ---- quantizer ------------------------------------------------------------------------------------------

def _check_quantize(w):
    wq, s = jq.mxfp4_quantize(w)
    K = w.shape[-1]
    code, byte = mo.quantize(_np(w).reshape(-1, K))
    assert wq.dtype == torch.int32 and s.dtype == torch.uint8 and wq.shape == w.shape[:-1] + (K // 8,) and s.shape == w.shape[:-1] + (K // 32,)
    assert np.array_equal(s.cpu().numpy().reshape(byte.shape), byte)
    assert np.array_equal(wq.cpu().numpy().view(np.uint32).reshape(len(byte), -1), mo.pack(code))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(32,), (1, 32), (3, 96), (257, 2080), (2, 5, 64), (1000, 1024)])
def test_quantize_matches_oracle(dtype, shape):
    _check_quantize(_rand(1, shape, dtype, 0.02))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantize_edges(dtype):
    """Zeros of both signs, ties of every neighbouring pair, saturation between 6 and 8, subnormals, the type's largest and
    smallest numbers, infinities and NaN."""
    t = torch.finfo(DT[dtype])
    ties = np.array([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.75, .125, .375, 5.5, 4.5, 6.5], np.float64)
    ties = np.concatenate([ties, -ties])[:32]
    blocks = [np.zeros(32), -np.zeros(32), ties[:32], ties * 2.0 ** -9, np.full(32, float(t.tiny)), np.full(32, float(t.smallest_normal)) * np.arange(32) / 32,
              np.full(32, float(t.max)), np.where(np.arange(32) == 9, float(t.max), 1.0), np.where(np.arange(32) == 31, np.inf, 1.0),
              np.where(np.arange(32) == 0, -np.inf, 0.0), np.where(np.arange(32) == 13, np.nan, 2.0), np.linspace(-1, 1, 32),
              np.where(np.arange(32) == 5, -7.9, 0.1), np.full(32, 2.0 ** -24), np.full(32, 2.0 ** -130)]
    w = torch.tensor(np.array(blocks), dtype=torch.float32).to(DT[dtype]).reshape(5, 96).cuda()
    _check_quantize(w)


@pytest.mark.gpu
def test_quantize_views():
    w = _rand(2, (65, 200), "bf16")
    _check_quantize(w[:, 3:195])                       # pitch and an unaligned start
    _check_quantize(w[:64].t()[:, :64])                # columns
    flat = _rand(3, (64 * 9 + 1,), "f16")
    _check_quantize(flat[1:].reshape(9, 64))           # contiguous, 2 bytes off
    _check_quantize(w[0, :64].expand(4, 64))
    wq, s = jq.mxfp4_quantize(w[:0, :64])
    assert wq.shape == (0, 8) and s.shape == (0, 2) and jq.mxfp4_dequantize(wq, s).shape == (0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_dequantize_every_code_and_scale(dtype):
    code = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    byte = np.arange(256, dtype=np.uint8)[:, None]
    words = mo.pack(code)
    out = jq.mxfp4_dequantize(torch.from_numpy(words.view(np.int32)).cuda(), torch.from_numpy(byte).cuda(), DT[dtype])
    want = torch.from_numpy(mo.values(words, byte)).to(torch.float32)            # exact up to 6 * 2^127
    assert torch.equal(torch.nan_to_num(out.cpu(), nan=7.0), torch.nan_to_num(want.to(DT[dtype]), nan=7.0))


@pytest.mark.gpu
def test_round_trip_of_representable_numbers():
    wq, s, v = _packed(4, (130, 1056))
    assert np.array_equal(_np(jq.mxfp4_dequantize(wq, s)), v)
    again = jq.mxfp4_quantize(jq.mxfp4_dequantize(wq, s, torch.float32))
    assert np.array_equal(_np(jq.mxfp4_dequantize(*again)), v)


# ---- products ---------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 16, 64), (1, 200, 96), (1, 4096, 2048), (2, 33, 288), (3, 129, 2080), (5, 64, 4096),
                                   (8, 1000, 320), (9, 15, 544), (16, 257, 2112), (1, 48, 14336), (16, 40, 8224), (7, 24, 12320), (1, 20, 36864),
                                   (2, 20, 36864), (1, 9, 40960)])
def test_matvec(M, N, K, dtype):
    wq, s, v = _packed(M + N + K, (N, K))
    x = _rand(K, (M, K), dtype)
    _close(jq.mxfp4_matmul(x, wq, s), _np(x), v, K)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 20011, 4128), (3, 10007, 4128), (8, 9999, 2112), (2, 40003, 2112)])
def test_matvec_over_many_tiles(M, N, K):
    """More row tiles per SM than the kernel puts aside before it adds them."""
    wq, s = jq.mxfp4_quantize(_rand(N, (N, K), "bf16", 0.02))
    x = _rand(K, (M, K), "bf16")
    w = jq.mxfp4_dequantize(wq, s, torch.float32).double()
    ref, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    y = jq.mxfp4_matmul(x, wq, s)
    tol = 2.0 ** -8 * ref.abs() + (K / 16 + 32) * 2.0 ** -23 * mag
    assert bool(((y.double() - ref).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 5])
def test_matvec_activations_of_very_different_size(M):
    """bf16 activations are scaled per block of 32, the largest to [2^14, 2^15), and rounded to f16, whose smallest step is 2^-24:
    an activation is off by at most 2^-25 of that scale, 2^-39 of the largest of its block.  Other blocks are not touched."""
    N, K = 64, 256
    wq, s, v = _packed(31, (N, K))
    x = _rand(32, (M, K), "bf16")
    x[:, 40] = 2.0 ** 100
    words = wq.clone()
    words[:, 5] = 0                                        # weights 40 .. 47 are zero: only the small activations count
    vz = v.copy()
    vz[:, 40:48] = 0
    x[:, 32:64] = torch.where(torch.arange(32, device="cuda") == 8, x[:, 32:64], x[:, 32:64] * 2.0 ** 72)
    xn = _np(x)
    for cols in (slice(0, 32), slice(32, 64)):
        one = torch.zeros_like(x)
        one[:, cols] = x[:, cols]
        one[:, 40] = x[:, 40]
        xo = _np(one)
        y = jq.mxfp4_matmul(one, words, s)
        ref, mag = xo @ vz.T, np.abs(xo) @ np.abs(vz).T
        blocks = np.abs(xo).reshape(M, -1, 32).max(-1)
        rounded = 2.0 ** -39 * (blocks[:, :, None] * np.abs(vz).reshape(N, -1, 32).sum(-1).T[None]).sum(1) if cols.start == 32 else 0.0
        assert np.all(np.abs(_np(y) - ref) <= 2.0 ** -8 * np.abs(ref) + (K / 16 + 32) * 2.0 ** -23 * mag + rounded)
    assert np.isfinite(xn).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(17, 1, 64), (17, 128, 96), (33, 130, 128), (61, 1000, 2048), (100, 257, 192), (200, 129, 2112),
                                   (256, 384, 512), (300, 72, 1088), (513, 513, 320), (40, 2880, 2880)])
def test_gemm(M, N, K, dtype):
    wq, s, v = _packed(M + N + K, (N, K))
    x = _rand(K, (M, K), dtype)
    _close(jq.mxfp4_matmul(x, wq, s), _np(x), v, K)


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 128, 64), (2, 200, 96), (16, 333, 256), (17, 128, 288), (33, 257, 1056), (128, 130, 512),
                                   (129, 64, 2080), (255, 129, 320), (256, 256, 1024), (300, 72, 4128), (520, 1000, 640),
                                   (5, 130, 8224), (128, 100, 4128), (130, 2100, 2112), (700, 5000, 288), (2100, 4101, 320),
                                   (1100, 9000, 1056), (2500, 4352, 288)])
def test_both_operands_quantized(M, N, K, out):
    wq, s, v = _packed(M + N + K, (N, K))
    xq, xs, xv = _packed(K, (M, K), 1.0)
    y = jq.mxfp4_matmul(xq, wq, s, x_scales=xs, dtype=DT[out])
    assert y.dtype == DT[out]
    _close(y, xv, v, K)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 8, 16, 40])
@pytest.mark.parametrize("K", [128, 4096])
def test_row_and_column_of_a_product_are_their_own(M, K):
    """One-hot activations pick single weights: every (row, k) goes where it belongs, in all three kernels."""
    N = 150
    wq, s, v = _packed(9, (N, K))
    hot = (np.arange(M) * 97 + 13) % K
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    x[torch.arange(M), torch.from_numpy(hot)] = 1.0
    assert np.array_equal(_np(jq.mxfp4_matmul(x, wq, s)), v[:, hot].T)
    xq, xs = jq.mxfp4_quantize(x)
    assert np.array_equal(_np(jq.mxfp4_matmul(xq, wq, s, x_scales=xs)), v[:, hot].T)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 16, 64])
def test_scales_over_the_whole_range(M):
    """Bytes from 0 to 254: single products, so nothing is lost in a sum; and a NaN block spoils its own row only.  In the
    tensor-core GEMM (here 16 and 64 rows) the weight enters in the activations' type, so a weight above its largest number is infinite
    -- 4 * 2^126 at byte 253 is 2^128, bf16 ends below it -- and the other, zero, activations make such a row NaN (0 * inf)."""
    K, N = 256, 255
    code = np.random.default_rng(3).integers(0, 16, (N, K)).astype(np.uint8)
    byte = np.repeat(np.arange(255, dtype=np.uint8)[:, None], K // 32, 1)
    words = mo.pack(code)
    v = mo.values(words, byte)
    wq, s = torch.from_numpy(words.view(np.int32)).cuda(), torch.from_numpy(byte).cuda()
    hot = (np.arange(M) * 37 + 5) % K
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    x[torch.arange(M), torch.from_numpy(hot)] = 1.0
    small = torch.from_numpy(np.abs(v[:, hot].T) < 2.0 ** -126)          # a subnormal product may be flushed

    def want(dtype, spoiled=None):
        w = torch.from_numpy(v).to(torch.float32).to(dtype)
        ref = w[:, torch.from_numpy(hot)].t().clone()
        if M <= 8:                                         # the mat-vec scales the sums: every weight is exact
            if spoiled is not None:
                ref[:, spoiled] = float("nan")
            return ref
        ref[:, w.isinf().any(1)] = float("nan")
        # every weight but the hot one meets a zero: a row whose only infinite weight is the hot one stays infinite
        for m, k in enumerate(hot):
            others = w.clone()
            others[:, k] = 0
            alone = w[:, k].isinf() & ~others.isinf().any(1)
            ref[m, alone] = w[alone, k]
        if spoiled is not None:
            ref[:, spoiled] = float("nan")
        return ref

    def same(y, ref):
        keep = ~small
        return torch.equal(y.isnan(), ref.isnan()) and torch.equal(torch.nan_to_num(y, nan=0.0)[keep], torch.nan_to_num(ref, nan=0.0)[keep])

    assert same(jq.mxfp4_matmul(x, wq, s).cpu(), want(torch.bfloat16))
    assert same(jq.mxfp4_matmul(x.half(), wq, s).cpu(), want(torch.float16))
    s2 = s.clone()
    s2[100, 3] = 255
    assert same(jq.mxfp4_matmul(x, wq, s2).cpu(), want(torch.bfloat16, 100))
    xq, xs = jq.mxfp4_quantize(x)
    y = jq.mxfp4_matmul(xq, wq, s2, x_scales=xs).cpu()
    assert bool(y[:, 100].isnan().all()) and not bool(y[:, :100].isnan().any()) and not bool(y[:, 101:].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 12, 50])
def test_activations_that_are_not_finite(M):
    """A row with an infinity or a NaN does not touch the others."""
    wq, s, v = _packed(5, (96, 192))
    x = _rand(6, (M, 192), "bf16")
    y = jq.mxfp4_matmul(x, wq, s)
    bad = x.clone()
    bad[M - 1, 17], bad[M - 1, 100] = float("inf"), float("nan")
    z = jq.mxfp4_matmul(bad, wq, s)
    assert torch.equal(z[:M - 1], y[:M - 1]) and bool(z[M - 1].isnan().all())


@pytest.mark.gpu
def test_matmul_views_and_leading_dimensions():
    wq, s, v = _packed(7, (72, 192))
    big = _rand(8, (64, 400), "bf16")
    for x in (big[:40, 8:200], big[:40, 3:195], big[:10, 8:200], big[:192, :40].t()[:, :64].repeat(1, 3), big[5:6, 16:208],
              big[3, :192].expand(33, 192), big[::2, 8:200]):
        _close(jq.mxfp4_matmul(x, wq, s), _np(x), v, 192)
    x = big[:60, :192].reshape(3, 20, 192)
    y = jq.mxfp4_matmul(x, wq, s)
    assert y.shape == (3, 20, 72)
    _close(y.reshape(60, 72), _np(x).reshape(60, 192), v, 192)
    assert jq.mxfp4_matmul(x[0, 0], wq, s).shape == (72,)
    assert jq.mxfp4_matmul(x[:0], wq, s).shape == (0, 20, 72)
    xq, xs = jq.mxfp4_quantize(x)
    assert jq.mxfp4_matmul(xq, wq, s, x_scales=xs).shape == (3, 20, 72)
    assert jq.mxfp4_matmul(xq[:0], wq, s, x_scales=xs[:0]).shape == (0, 20, 72)
    wide = torch.zeros((72, 30), dtype=torch.int32, device="cuda")
    wide[:, 3:27] = wq
    assert torch.equal(jq.mxfp4_matmul(x, wide[:, 3:27], s), y)
    assert torch.equal(jq.mxfp4_matmul(x, wq.view(torch.uint32), s), y)


# ---- experts ------------------------------------------------------------------------------------------------

def _experts_close(y, x, idx, v, k):
    flat = idx.reshape(-1).cpu().numpy()
    K = x.shape[1]
    xn = _np(x)
    for e in np.unique(flat):
        at = np.nonzero(flat == e)[0]
        if 0 <= e < len(v):
            _close(y[torch.from_numpy(at).cuda()], xn[at // k], v[e], K)
        else:
            assert not bool(y[torch.from_numpy(at).cuda()].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,k,E,N,K", [(1, 1, 1, 1, 32), (1, 8, 16, 96, 256), (7, 3, 5, 33, 96), (3, 21, 8, 200, 128), (16, 4, 8, 136, 192),
                                       (50, 4, 8, 72, 320), (33, 2, 4, 100, 96), (300, 2, 3, 257, 128), (1, 64, 9, 40, 64), (700, 1, 2, 64, 64)])
def test_gather(T, k, E, N, K, dtype):
    wq, s, v = _packed(T + E, (E, N, K))
    x = _rand(T, (T, K), dtype)
    idx = torch.from_numpy(np.random.default_rng(T).integers(0, E, (T, k))).int().cuda()
    idx[0, 0] = E - 1
    y = jq.mxfp4_gather_matmul(x, wq, s, rhs_indices=idx)
    assert y.shape == (T * k, N)
    _experts_close(y, x, idx, v, k)
    bank = jq.MXFP4ExpertBank(wq, s)
    assert torch.equal(jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx.long()), y)
    lhs = torch.arange(T * k, device="cuda") // k
    assert torch.equal(jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx.reshape(-1), lhs_indices=lhs, sorted_indices=True), y)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [12, 300])
def test_gather_with_experts_elsewhere_and_all_on_one(pairs):
    E, N, K = 6, 80, 128
    wq, s, v = _packed(1, (E, N, K))
    x = _rand(2, (pairs, K), "bf16")
    idx = torch.from_numpy(np.random.default_rng(3).integers(-2, E + 2, pairs)).int().cuda()
    _experts_close(jq.mxfp4_gather_matmul(x, wq, s, rhs_indices=idx), x, idx, v, 1)
    bad = x.clone()
    bad[:, 3] = float("nan")                               # not even the rows of pairs without an expert take it over
    y = jq.mxfp4_gather_matmul(bad, wq, s, rhs_indices=idx)
    away = (idx < 0) | (idx >= E)
    assert not bool(y[away].any()) and bool(y[~away].isnan().all())
    for e in (0, 5, -1, E):
        _experts_close(jq.mxfp4_gather_matmul(x, wq, s, rhs_indices=torch.full_like(idx, e)), x, torch.full_like(idx, e), v, 1)
    assert jq.mxfp4_gather_matmul(x[:0], wq, s, rhs_indices=idx[:0]).shape == (0, N)
    far = idx.long().clamp(0, E - 1)
    far[::3] += 2 ** 32                                    # an expert of the bank in its low 32 bits
    y = jq.mxfp4_gather_matmul(x, wq, s, rhs_indices=far)
    assert not bool(y[::3].any()) and torch.equal(y[1::3], jq.mxfp4_gather_matmul(x, wq, s, rhs_indices=idx.clamp(0, E - 1))[1::3])
    lhs = torch.arange(pairs, device="cuda") - 1           # -1 names the first row
    y = jq.mxfp4_gather_matmul(x, wq, s, rhs_indices=idx, lhs_indices=lhs)
    _experts_close(y, x[lhs.clamp(min=0)], idx, v, 1)


def _silu(g):
    return g / (1.0 + np.exp(-g))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,k,limit,shared", [(1, 4, 0.0, False), (5, 4, 0.5, False), (40, 4, 0.0, True), (150, 3, 0.5, False)])
def test_router_and_moe_layer(T, k, limit, shared, dtype):
    """A routed layer as it is used: route_topk, then moe_layer over MXFP4 banks, few tokens and many.  The rounding of the
    gate and up rows (few tokens), of h and of the expert rows is half a step each of magnitudes that the bound carries
    through: three half steps of sum |h| |w_down| plus one of the output, times 2 for the slope of the SwiGLU."""
    E, H, I = 16, 256, 192
    x = _rand(T, (T, H), dtype)
    logits = _rand(T + 1, (T, E))
    bias = _rand(3, (E,), scale=0.1)
    gq, gs, gv = _packed(11, (E, I, H), 0.1)
    uq, us, uv = _packed(12, (E, I, H), 0.1)
    dq, ds, dv = _packed(13, (E, H, I), 0.1)
    idx, w = jq.route_topk(logits, k, score="sigmoid", bias=bias, groups=4, groups_kept=2, scale=2.0)
    ri, rw = mo.route(_np(logits), k, "sigmoid", _np(bias), 4, 2, 2, True, 2.0)
    assert np.array_equal(idx.cpu().numpy(), ri)
    sh = tuple(jq.JANGLinear.from_float(_rand(20 + i, shape, dtype, 0.1), bits=8, group_size=64)
               for i, shape in enumerate(((I, H), (I, H), (H, I)))) if shared else None
    banks = (jq.MXFP4ExpertBank(gq, gs), jq.MXFP4ExpertBank(uq, us), jq.MXFP4ExpertBank(dq, ds))
    out = jq.moe_layer(x, idx, w, *banks, swiglu_limit=limit, shared=sh)
    f32 = jq.moe_layer(x, idx, w, *banks, swiglu_limit=limit, shared=sh, out_f32=True)
    xn = _np(x)

    def expert(g, u, wt):
        g, u = (np.minimum(g, limit), np.clip(u, -limit, limit)) if limit else (g, u)
        return _silu(g) * u * wt

    ref, mag = np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        for j in range(k):
            e = ri[t, j]
            g, u = gv[e] @ xn[t], uv[e] @ xn[t]
            h = expert(g, u, rw[t, j])
            # what a half step of g and of u can do to h: |silu'| <= 1.1
            spread = np.abs(h) + (np.abs(g) + np.abs(_silu(g))) * np.abs(u) * rw[t, j] * 1.1
            ref[t] += dv[e] @ h
            mag[t] += np.abs(dv[e]) @ spread + np.abs(dv[e] @ h)
    if shared:
        sg, su, sd = (_np(jq.dequantize(m.weight, m.scales, m.biases, 64, 8, dtype=torch.float32)) for m in sh)
        g, u = xn @ sg.T, xn @ su.T
        h = expert(g, u, 1.0)
        ref += h @ sd.T
        mag += 2 * (np.abs(h) + (np.abs(g) + np.abs(_silu(g))) * np.abs(u)) @ np.abs(sd).T + np.abs(h @ sd.T) \
            + np.abs(h) @ np.abs(sd).T + np.abs(xn) @ np.abs(sg).T.max(1, keepdims=True)
    step = torch.finfo(DT[dtype]).eps / 2
    for y in (out, f32):
        err = np.abs(_np(y) - ref)
        tol = 3 * step * mag + step * np.abs(ref) + 1e-4 * mag
        assert np.all(err <= tol), float((err / tol).max())
    assert f32.dtype == torch.float32 and out.dtype == DT[dtype]
    # an expert-parallel shard: the two halves' parts add up
    halves = [jq.moe_layer(x, idx, w, *(jq.MXFP4ExpertBank(b.weight[i:i + 8], b.scales[i:i + 8]) for b in banks), swiglu_limit=limit,
                           expert_base=i, out_f32=True) for i in (0, 8)]
    whole = jq.moe_layer(x, idx, w, *banks, swiglu_limit=limit, out_f32=True)
    torch.testing.assert_close(halves[0] + halves[1], whole, rtol=1e-5, atol=1e-5)


# ---- streams, graphs, refusals --------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 120])
def test_captured_layer_replays_on_new_inputs(T):
    E, H, I, k = 8, 128, 64, 2
    banks = [jq.MXFP4ExpertBank.from_float(_rand(i, shape, "bf16", 0.1)) for i, shape in enumerate(((E, I, H), (E, I, H), (E, H, I)))]
    x, logits = _rand(1, (T, H), "bf16"), _rand(2, (T, E))

    def step():
        idx, w = jq.route_topk(logits, k, groups=4, groups_kept=2)
        y = jq.moe_layer(x, idx, w, *banks)
        q, s = jq.mxfp4_quantize(y)
        return jq.mxfp4_matmul(q, banks[0].weight[0], banks[0].scales[0], x_scales=s), y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
        for seed in (5, 6):
            x.copy_(_rand(seed, (T, H), "bf16"))
            logits.copy_(_rand(seed + 10, (T, E)))
            graph.replay()
            want = step()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.current_stream().wait_stream(side)
    jq._lib.check(jq._lib.load().jq_device_status())


@pytest.mark.gpu
def test_bank_tables_are_there_for_other_streams():
    w, s = jq.mxfp4_quantize(torch.zeros((5, 8, 64), device="cuda"))
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)                        # some tens of milliseconds of the current stream
    bank = jq.MXFP4ExpertBank(w, s)
    with torch.cuda.stream(other):
        codes, scales = bank.codes_tab.cpu(), bank.scales_tab.cpu()
    assert codes.tolist() == [w.data_ptr() + e * 8 * 32 for e in range(5)]
    assert scales.tolist() == [s.data_ptr() + e * 8 * 2 for e in range(5)]
    graph, x, idx = torch.cuda.CUDAGraph(), torch.ones((70, 64), device="cuda", dtype=torch.bfloat16), torch.zeros((70, 1), dtype=torch.int32, device="cuda")
    with torch.cuda.graph(graph):                        # stacked codes, and a bank, inside a capture
        y = jq.mxfp4_gather_matmul(x, w, s, rhs_indices=idx)
        z = jq.mxfp4_gather_matmul(x, jq.MXFP4ExpertBank(w, s), rhs_indices=idx)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(z, y)


@pytest.mark.gpu
def test_two_streams_at_once():
    wq, s, v = _packed(3, (640, 512))
    xs = [_rand(i, (m, 512), "bf16") for i, m in enumerate((1, 12, 70, 300))]
    want = [jq.mxfp4_matmul(x, wq, s) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(jq.mxfp4_matmul(x, wq, s))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 4]) for i, y in enumerate(got))


@pytest.mark.gpu
def test_refusals():
    z = lambda shape, dt: torch.zeros(shape, dtype=dt, device="cuda")          # noqa: E731
    wq, s = z((8, 16), torch.int32), z((8, 4), torch.uint8)
    x = z((2, 128), torch.bfloat16)
    bank = jq.MXFP4ExpertBank(z((4, 8, 16), torch.int32), z((4, 8, 4), torch.uint8))
    idx = z((2, 2), torch.int32)
    calls = [lambda: jq.mxfp4_quantize(z((4, 33), torch.float32)), lambda: jq.mxfp4_quantize(z((4, 0), torch.float32)),
             lambda: jq.mxfp4_quantize(z((4, 32), torch.float64)), lambda: jq.mxfp4_quantize(z((), torch.float32)),
             lambda: jq.mxfp4_dequantize(wq, s[:, :3]), lambda: jq.mxfp4_dequantize(wq[:, :3], s), lambda: jq.mxfp4_dequantize(wq.float(), s),
             lambda: jq.mxfp4_dequantize(wq, s.int()), lambda: jq.mxfp4_dequantize(wq, s, torch.float64),
             lambda: jq.mxfp4_dequantize(wq[:, :0], s[:, :0]),
             lambda: jq.mxfp4_matmul(x[:, :96], wq, s), lambda: jq.mxfp4_matmul(x.float(), wq, s), lambda: jq.mxfp4_matmul(x, wq[None], s[None]),
             lambda: jq.mxfp4_matmul(x, wq, s, dtype=torch.float32), lambda: jq.mxfp4_matmul(x.cpu(), wq, s),
             lambda: jq.mxfp4_matmul(z((2, 36896), torch.bfloat16), z((4, 4612), torch.int32), z((4, 1153), torch.uint8)),
             lambda: jq.mxfp4_matmul(wq, wq, s), lambda: jq.mxfp4_matmul(wq[:, :12], wq, s, x_scales=s[:, :3]),
             lambda: jq.mxfp4_matmul(wq, wq, s, x_scales=s, dtype=torch.float64), lambda: jq.mxfp4_matmul(x, wq, s, x_scales=s),
             lambda: jq.MXFP4ExpertBank(wq, s), lambda: jq.MXFP4ExpertBank(bank.weight[:0], bank.scales[:0]),
             lambda: jq.mxfp4_gather_matmul(x, bank), lambda: jq.mxfp4_gather_matmul(x, bank.weight, rhs_indices=idx),
             lambda: jq.mxfp4_gather_matmul(x[:, :64], bank, rhs_indices=idx), lambda: jq.mxfp4_gather_matmul(x.float(), bank, rhs_indices=idx),
             lambda: jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx[:1].reshape(-1)[:1]),
             lambda: jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx, lhs_indices=idx[0]),
             lambda: jq.moe_layer(x, idx, idx.float(), bank, bank, bank), lambda: jq.moe_layer(x, idx[:, :0], idx[:, :0].float(), bank, bank, bank),
             lambda: jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx.float()), lambda: jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx[:, :0]),
             lambda: jq.mxfp4_gather_matmul(x[:0], bank, rhs_indices=idx, lhs_indices=idx),
             lambda: jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx, lhs_indices=idx.float()),
             lambda: jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx.to(torch.uint64)),
             lambda: jq.moe_layer(x, idx, idx.float(), bank, bank, None), lambda: jq.moe_layer(x, idx, idx.float(), bank, bank, bank, return_slots=True)]
    for i, call in enumerate(calls):
        with pytest.raises(JangqError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(ValueError):
        jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx, sorted_indices=True)


def test_cpu_tensors_are_refused():
    for call in (lambda: jq.mxfp4_quantize(torch.zeros(4, 64)), lambda: jq.mxfp4_dequantize(torch.zeros(4, 8, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.uint8)),
                 lambda: jq.mxfp4_matmul(torch.zeros(4, 64), torch.zeros(4, 8, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.uint8)),
                 lambda: jq.MXFP4ExpertBank(torch.zeros(2, 4, 8, dtype=torch.int32), torch.zeros(2, 4, 2, dtype=torch.uint8))):
        with pytest.raises(JangqError):
            call()


def test_argument_checks_need_no_gpu():
    lib, L = jq._lib.load(), jq._lib
    assert lib.jq_mxfp4_quantize(None, L.JQ_F32, 4, 33, None, None, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_quantize(None, L.JQ_F32, 4, 64, None, None, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_quantize(None, 9, 4, 64, None, None, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_dequantize(None, None, -1, 64, None, L.JQ_F32, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_gemv(None, L.JQ_BF16, 17, 64, None, None, 4, 64, None, 4, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_gemv(16, L.JQ_F32, 1, 64, 16, 16, 4, 64, 16, 4, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_gemv(16, L.JQ_BF16, 1, 60, 16, 16, 4, 64, 16, 4, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_gemm(16, L.JQ_BF16, 20, 96, 16, 16, 4, 96, 16, 4, None) == L.JQ_EUNSUPPORTED
    assert lib.jq_mxfp4_gather_gemv(16, L.JQ_BF16, 64, 0, 16, 1, 16, 16, 1, 0, 4, 64, 16, 4, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_gather_gemv(16, L.JQ_BF16, 64, 1, 16, 1 << 17, 16, 16, 1, 0, 4, 64, 16, 4, None) == L.JQ_EUNSUPPORTED
    assert lib.jq_mxfp4_gemm4(None, None, 4, None, None, 4, 64, None, L.JQ_BF16, 4, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_gemm4(8, 16, 4, 16, 16, 4, 64, 16, L.JQ_BF16, 4, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_moe_gemm(16, L.JQ_BF16, 4, 64, 16, 16, 16, 16, 1, 256, 16, 16, 4, 64, None, None, 16, 4, None) == L.JQ_EINVAL
    assert lib.jq_mxfp4_moe_gemm(16, L.JQ_BF16, 4, 64, 16, 16, 16, 16, 1, 192, 16, 16, 4, 64, 16, None, 16, 4, None) == L.JQ_EINVAL
    assert lib.jq_moe_route_topk(16, L.JQ_F32, 8, 1, 8, 2, 2, None, 1, 1, 1, 1, 1.0, 16, 16, None) == L.JQ_EINVAL
