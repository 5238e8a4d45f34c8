"""Microscaled 4-bit floating point (OCP MXFP4) beside the affine codec: quantizer, products, experts' products.

    mxfp4_quantize / mxfp4_dequantize   <-> quantize / dequantize
    mxfp4_matmul                        <-> quantized_matmul; with x_scales both operands are MXFP4
    mxfp4_gather_matmul, MXFP4ExpertBank <-> gather_qmm, ExpertBank

A tensor is a pair: codes torch.int32 [.., K/8] (eight e2m1 numbers per word, the first in the lowest bits, the affine
codec's 4-bit layout) and scales torch.uint8 [.., K/32], the power of two 2^(byte - 127) of 32 neighbouring numbers.
The reference writes such bundles with its MXFP4 converters and runs them through mx.quantized_matmul.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import JangqError

BLOCK = 32
# Pairs from which the grouped product runs, as gather_qmm.  A mat-vec per pair takes about 4 us + pairs * (expert bytes / 4.6 TB/s),
# the sort, the row gather and the product 12 us + 0.26 us per k-block and round of tiles, so the sizes at which they meet differ:
# 64 pairs of 8 experts of 2048x4096 66.8 us one by one and 29.1 grouped (they meet at 24), of 32 of 1024x2048 20.5 and 29.6 (at 100), of 128
# of 768x2048 17.3 and 37.3 (at 320), of 512 of 512x2048 13 and 31.
SORT_THRESHOLD = 64
# Rows that the mat-vec takes in one launch (their activations in shared memory: rows * K up to MXFP4_GEMV_MAX_K).  Beyond,
# every weight is read again, and the tensor-core GEMM is faster: bf16, 8 rows of 14336x4096 16.8 us here, 20.4 there, 9 rows 29
# and 20; 8 rows of 4096x4096 9.5 and 9.3, of 2048x2048 5.8 and 6.3, 9 rows 10 and 6.4; 2 rows of 4096x14336 15.3 and 19.0, 4 rows
# 29 and 19; f16, 8 rows of 14336x4096 14.1 and 17.3.
MATVEC_ROWS = 8


# A small product is a few microseconds of kernel, so the checks below take the short way where there is one: no slices and
# no reshapes that change nothing, and new_empty, which is cheaper than torch.empty with a device.

def _check_pair(wq: torch.Tensor, scales: torch.Tensor, what: str = "codes"):
    """int32 codes and uint8 scales of one shape, contiguous and aligned for the kernels -> (codes, scales, K)."""
    if wq.dtype is torch.uint32:
        wq = wq.view(torch.int32)
    if wq.dtype is not torch.int32 or scales.dtype is not torch.uint8:
        raise JangqError(_lib.JQ_EINVAL, f"{what} must be int32/uint32 and scales uint8, got {wq.dtype} and {scales.dtype}")
    shape = wq.shape
    words = shape[-1] if shape else 0
    if words == 0 or words % 4:
        raise JangqError(_lib.JQ_EINVAL, f"{what} of shape {tuple(shape)} do not hold whole blocks of {BLOCK}")
    if scales.shape != shape[:-1] + (words // 4,):
        raise JangqError(_lib.JQ_EINVAL, f"scales shape {tuple(scales.shape)} does not match {what} {tuple(shape)}: one byte "
                                         f"per {BLOCK} numbers")
    if not wq.is_contiguous() or wq.data_ptr() % 16:
        wq = _aligned(wq)
    if not scales.is_contiguous() or scales.data_ptr() % 16:
        scales = _aligned(scales)
    return wq, scales, words * 8


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def rows_ok(x: torch.Tensor) -> torch.Tensor:
    """x [M, K] itself where the kernels take its rows (16-byte aligned, unit stride), else a copy."""
    M, K = x.shape
    if x.stride(1) == 1 and x.data_ptr() % 16 == 0:
        if M == 1:           # the pitch of a single row is whatever the view it came from had and says nothing
            return x if x.stride(0) == K else x.as_strided((1, K), (K, 1))
        if x.stride(0) % 8 == 0 and x.stride(0) >= K:
            return x
    return _aligned(x)


def mxfp4_quantize(w: torch.Tensor):
    """MXFP4 along the last axis (a multiple of 32) -> (codes int32 [.., K/8], scales uint8 [.., K/32]).

    Per 32 numbers the scale is 2^(floor(log2(max |w|)) - 2), not below 2^-127; numbers go to the nearest of
    0 .5 1 1.5 2 3 4 6 times the scale, ties to the even code, 6 and above to 6.  A block with an infinity or a NaN gets
    scale byte 255 and dequantizes to NaN.  w: float32, float16 or bfloat16."""
    dev = _lib.require_cuda(w)
    lib = _lib.load()
    if w.dim() < 1 or w.shape[-1] % BLOCK or w.shape[-1] == 0:
        raise JangqError(_lib.JQ_EINVAL, f"mxfp4_quantize expects rows of whole blocks of {BLOCK}, got {tuple(w.shape)}")
    dt = _lib.dtype_id(w.dtype)
    K = w.shape[-1]
    if not w.is_contiguous() or w.data_ptr() % 16:
        w = _aligned(w)
    lead = w.shape[:-1]
    wq = w.new_empty(lead + (K // 8,), dtype=torch.int32)
    scales = w.new_empty(lead + (K // BLOCK,), dtype=torch.uint8)
    with _lib.on_device(dev):
        _lib.check(lib.jq_mxfp4_quantize(w.data_ptr(), dt, w.numel() // K, K, wq.data_ptr(), scales.data_ptr(),
                                         _lib.stream_ptr(dev)))
    return wq, scales


def mxfp4_dequantize(wq: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The numbers a packed pair stands for -> [.., K], rounded once to `dtype` (exact in bfloat16 and float32 but for
    2^128 and above, which mxfp4_quantize does not give)."""
    dev = _lib.require_cuda(wq, scales)
    lib = _lib.load()
    wq, scales, K = _check_pair(wq, scales)
    out = wq.new_empty(wq.shape[:-1] + (K,), dtype=dtype)
    with _lib.on_device(dev):
        _lib.check(lib.jq_mxfp4_dequantize(wq.data_ptr(), scales.data_ptr(), out.numel() // K, K, out.data_ptr(),
                                           _lib.dtype_id(dtype), _lib.stream_ptr(dev)))
    return out


def mxfp4_matmul(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, x_scales: torch.Tensor | None = None,
                 dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[.., N] = x[.., K] . deq(w, scales)[N, K]^T with float32 sums.

    x bfloat16 or float16: few rows run the mat-vec kernel, more the tensor-core GEMM; the output has x's type.  In
    the GEMM the weight enters in it (exact in bfloat16, but infinite from 2^128 on; in float16 rounded once, and
    beyond 65504 infinite); the mat-vec rounds bfloat16 activations below 2^-29 of the largest of their block of 32, by
    less than 2^-39 of it.
    x int32 codes [.., K/8] with x_scales uint8 [.., K/32] (mxfp4_quantize of the activations): both operands go to the
    tensor cores in 4 bits; the output type is `dtype` (bfloat16 by default)."""
    dev = _lib.require_cuda(x, w, scales, x_scales)
    lib = _lib.load()
    w, scales, K = _check_pair(w, scales, "weight codes")
    if w.dim() != 2:
        raise JangqError(_lib.JQ_EINVAL, f"weight must be 2-D [N, K/8], got {tuple(w.shape)}")
    N = w.shape[0]
    if x_scales is not None:
        x, x_scales, kx = _check_pair(x, x_scales, "activation codes")
        if kx != K:
            raise JangqError(_lib.JQ_EINVAL, f"x has {kx} features, weight expects {K}")
        y = x.new_empty(x.shape[:-1] + (N,), dtype=dtype or torch.bfloat16)
        with _lib.on_device(dev):
            _lib.check(lib.jq_mxfp4_gemm4(x.data_ptr(), x_scales.data_ptr(), x.numel() // (K // 8), w.data_ptr(),
                                          scales.data_ptr(), N, K, y.data_ptr(), _lib.dtype_id(y.dtype), N, _lib.stream_ptr(dev)))
        return y
    if x.dtype is not torch.bfloat16 and x.dtype is not torch.float16:
        raise JangqError(_lib.JQ_EINVAL, f"activations must be bfloat16 or float16 (or MXFP4 codes with x_scales), got {x.dtype}")
    if dtype is not None and dtype != x.dtype:
        raise JangqError(_lib.JQ_EUNSUPPORTED, f"the output of 16-bit activations has their type, {x.dtype}")
    xshape = x.shape
    if not xshape or xshape[-1] != K:
        raise JangqError(_lib.JQ_EINVAL, f"x of shape {tuple(xshape)} does not have the weight's {K} features")
    y = x.new_empty(xshape[:-1] + (N,))
    x2 = rows_ok(x if len(xshape) == 2 else x.reshape(-1, K))
    M, ld = x2.shape[0], x2.stride(0)
    dt, xp, yp, wp, sp = _lib.dtype_id(x.dtype), x2.data_ptr(), y.data_ptr(), w.data_ptr(), scales.data_ptr()
    with _lib.on_device(dev):
        st = _lib.stream_ptr(dev)
        if K % 64 == 0 and (M > MATVEC_ROWS or M * K > _lib.MXFP4_GEMV_MAX_K):
            _lib.check(lib.jq_mxfp4_gemm(xp, dt, M, ld, wp, sp, N, K, yp, N, st))
        else:
            # An odd number of blocks is the mat-vec's, 16 rows at a time: every 8 rows read the weights again (4096x2080: 64 rows 57 us,
            # 2048 rows 1800; 4096x2112 8.9 and 34).
            for m0 in range(0, M, _lib.QGEMV_MAX_M):
                _lib.check(lib.jq_mxfp4_gemv(xp + 2 * m0 * ld, dt, min(_lib.QGEMV_MAX_M, M - m0), ld, wp, sp, N, K,
                                             yp + 2 * m0 * N, N, st))
    return y


class MXFP4ExpertBank:
    """MXFP4 weights of E experts for one projection: `weight` int32/uint32 [E, N, K/8], `scales` uint8 [E, N, K/32].
    The device pointer tables of the grouped products are built once (one_call: for a product that follows at once, by it)."""

    def __init__(self, weight: torch.Tensor, scales: torch.Tensor, one_call: bool = False):
        self.device = _lib.require_cuda(weight, scales)
        if weight.dim() != 3:
            raise JangqError(_lib.JQ_EINVAL, f"stacked expert weight must be [E, N, K/8], got {tuple(weight.shape)}")
        self.weight, self.scales, self.K = _check_pair(weight, scales, "expert codes")
        self.E, self.N = self.weight.shape[:2]
        if self.E < 1 or self.N < 1:
            raise JangqError(_lib.JQ_EINVAL, f"a bank holds at least one row of one expert, got {tuple(weight.shape)}")
        # The pointers are complete when the constructor returns: a product on another stream that does not wait for this one would
        # read wrong numbers from weights on their way, but fault on pointers.  A capture cannot wait, and a table that it fills holds
        # nothing until a replay; a bank made in one leaves the tables to the products, each of which builds its own.
        self._tables = None
        with _lib.on_device(self.device):
            if not one_call and not torch.cuda.is_current_stream_capturing():
                self._tables = tuple(t.to(self.device) for t in self._pointers("cpu"))

    def _pointers(self, device):
        """int64 tables of the experts' codes and scales."""
        return tuple(torch.arange(p, p + self.E * step, step, dtype=torch.int64, device=device)
                     for p, step in ((self.weight.data_ptr(), self.N * self.K // 2), (self.scales.data_ptr(), self.N * self.K // BLOCK)))

    def tables(self):
        """Device pointer tables (codes, scales) for work on the current stream; the caller holds them until it is launched."""
        return self._tables or self._pointers(self.device)

    @property
    def codes_tab(self) -> torch.Tensor:
        return self.tables()[0]

    @property
    def scales_tab(self) -> torch.Tensor:
        return self.tables()[1]

    @classmethod
    def from_float(cls, w: torch.Tensor) -> "MXFP4ExpertBank":
        """Quantize float experts [E, N, K] on the GPU (mxfp4_quantize)."""
        return cls(*mxfp4_quantize(w))

    @property
    def gemm_ok(self) -> bool:
        """Shapes the tensor-core grouped product takes."""
        return self.K % 64 == 0

    def use_gemm(self, pairs: int) -> bool:
        """The grouped product, not a mat-vec per pair: many pairs, or rows too long for the mat-vec (and no more experts
        than the sort in front of it takes)."""
        return self.gemm_ok and self.E <= _lib.MOE_SORT_MAX_EXPERTS and (pairs >= SORT_THRESHOLD or self.K > _lib.MXFP4_GEMV_MAX_K)


def _check_integers(idx: torch.Tensor, what: str):
    if idx.is_floating_point() or idx.is_complex() or idx.dtype in (torch.bool, torch.uint64):
        raise JangqError(_lib.JQ_EINVAL, f"{what} must be integers of up to 64 bits with a sign, got {idx.dtype}")


def expert_ids(idx: torch.Tensor, base: int, experts: int) -> torch.Tensor:
    """Contiguous int32 expert ids of the pairs; ids beyond 32 bits stay outside [base, base + experts)."""
    if idx.dtype is torch.int32:
        return idx if idx.is_contiguous() else idx.contiguous()
    if idx.dtype is torch.int64:
        idx = idx.clamp(base - 1, base + experts)
    else:
        _check_integers(idx, "expert indices")
    return idx.to(torch.int32).contiguous()


def expert_gemv(x: torch.Tensor, x_div: int, pair_expert: torch.Tensor, bank: MXFP4ExpertBank, expert_base: int = 0) -> torch.Tensor:
    """y[p] = deq(W[pair_expert[p] - expert_base]) . x[p // x_div], one mat-vec per pair; rows of experts outside the bank
    are zero."""
    lib = _lib.load()
    P = pair_expert.numel()
    N, K, ld = bank.N, bank.K, x.stride(0)
    y = x.new_empty((P, N))
    dt, xp, ip, yp = _lib.dtype_id(x.dtype), x.data_ptr(), pair_expert.data_ptr(), y.data_ptr()
    wp, sp, st = bank.weight.data_ptr(), bank.scales.data_ptr(), _lib.stream_ptr(x.device)
    step = max(1, 32768 // x_div) * x_div             # pairs of one launch, those of whole tokens
    for p0 in range(0, P, step):
        _lib.check(lib.jq_mxfp4_gather_gemv(xp + 2 * (p0 // x_div) * ld, dt, ld, x_div, ip + 4 * p0, min(step, P - p0), wp, sp,
                                            bank.E, expert_base, N, K, yp + 2 * p0 * N, N, st))
    return y


def expert_gemm(x_sorted: torch.Tensor, sp, bank: MXFP4ExpertBank, scatter: bool = False) -> torch.Tensor:
    """The grouped product over expert-sorted rows (moe.SortedPairs); scatter=True stores the rows where their pairs stand,
    and zeros for the pairs of no expert of the bank."""
    lib = _lib.load()
    codes, scales = bank.tables()
    y = x_sorted.new_empty((x_sorted.shape[0], bank.N))
    _lib.check(lib.jq_mxfp4_moe_gemm(x_sorted.data_ptr(), _lib.dtype_id(x_sorted.dtype), sp.n, x_sorted.stride(0),
                                     sp.offsets.data_ptr(), sp.tile_expert.data_ptr(), sp.tile_row0.data_ptr(),
                                     sp.num_tiles.data_ptr(), sp.max_tiles, sp.tile_m, codes.data_ptr(),
                                     scales.data_ptr(), bank.N, bank.K, sp.order.data_ptr() if scatter else None,
                                     sp.inv.data_ptr() if scatter else None, y.data_ptr(), bank.N,
                                     _lib.stream_ptr(x_sorted.device)))
    return y


def mxfp4_gather_matmul(x: torch.Tensor, w, scales: torch.Tensor | None = None, rhs_indices: torch.Tensor | None = None,
                        lhs_indices: torch.Tensor | None = None, sorted_indices: bool = False) -> torch.Tensor:
    """y[r] = x[lhs[r]] . deq(w[rhs[r]])^T for stacked MXFP4 experts w [E, N, K/8], scales [E, N, K/32] (or an
    MXFP4ExpertBank): gather_qmm's call shape, indices and result [R, N] (x [R0, K]; rhs_indices [R] or [T, k]; without
    lhs_indices row r of x is used when R0 == R, row r // k when rhs is [T, k] with R0 == T).  Indices outside the bank
    give rows of zeros; lhs indices outside x take its first or last row.  Below 64 rows one mat-vec per row, above that the grouped tensor-core product."""
    if rhs_indices is None:
        raise JangqError(_lib.JQ_EINVAL, "mxfp4_gather_matmul needs rhs_indices")
    if sorted_indices and lhs_indices is None:
        raise ValueError("sorted_indices=True requires lhs_indices")
    if not isinstance(w, MXFP4ExpertBank) and scales is None:
        raise JangqError(_lib.JQ_EINVAL, "mxfp4_gather_matmul needs scales with stacked codes")
    bank = w if isinstance(w, MXFP4ExpertBank) else MXFP4ExpertBank(w, scales, one_call=True)
    dev = _lib.require_cuda(x, rhs_indices, lhs_indices, bank.weight)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise JangqError(_lib.JQ_EINVAL, f"activations must be bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] != bank.K:
        raise JangqError(_lib.JQ_EINVAL, f"x of shape {tuple(x.shape)} does not have the experts' {bank.K} features")
    x2 = x if x.dim() == 2 else x.reshape(-1, bank.K)
    k = rhs_indices.shape[-1] if rhs_indices.dim() == 2 else 1
    R = rhs_indices.numel()
    rhs = expert_ids(rhs_indices, 0, bank.E)
    if lhs_indices is not None:
        _check_integers(lhs_indices, "lhs_indices")
        lhs = lhs_indices.reshape(-1).to(torch.int64)
        if lhs.numel() != R or (x2.shape[0] == 0 and R > 0):
            raise JangqError(_lib.JQ_EINVAL, "lhs_indices and rhs_indices differ in length, or there are no rows of x")
        # an index outside x names its first or last row: a read out of range would end the process
        x2, x_div = x2.index_select(0, lhs.clamp(0, max(x2.shape[0] - 1, 0))), 1
    elif x2.shape[0] == R:
        x_div = 1
    elif rhs_indices.dim() == 2 and x2.shape[0] == rhs_indices.shape[0] and k > 0:
        x_div = k
    else:
        raise JangqError(_lib.JQ_EINVAL, f"cannot match {x2.shape[0]} rows of x with {R} indices")
    if R == 0:
        return x.new_empty((0, bank.N))
    x2 = rows_ok(x2)
    with _lib.on_device(dev):
        if not bank.use_gemm(R):
            return expert_gemv(x2, x_div, rhs, bank)
        from . import moe
        sp = moe.SortedPairs(rhs, bank.E, tile_m=_lib.MOE_GEMM_TILE_M)
        return expert_gemm(moe._gather_rows(x2, sp, x_div), sp, bank, scatter=True)
