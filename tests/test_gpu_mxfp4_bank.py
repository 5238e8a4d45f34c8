"""Pointer tables and sizes of MXFP4 expert banks."""
import numpy as np
import pytest
import torch

import jangq_b200 as jq

from oracle import mxfp4_oracle as mo


def _rand(seed, shape, scale=1.0):
    return torch.tensor(np.random.default_rng(seed).standard_normal(shape) * scale, dtype=torch.float32).to(torch.bfloat16).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [False, True])
def test_bank_made_in_a_capture_before_and_after_its_replay(layer):
    """The products take the bank's pointers from no table that only a replay fills."""
    E, N, K, T = 6, 64, 128, 80
    w, s = jq.mxfp4_quantize(_rand(1, (E, N, K), 0.1))
    w2, s2 = jq.mxfp4_quantize(_rand(2, (E, K, N), 0.1))
    x, idx = _rand(3, (T, K)), torch.arange(T, device="cuda", dtype=torch.int32).reshape(T, 1) % E
    wt = torch.ones((T, 1), device="cuda")

    def use(bank, down):
        if layer:
            return jq.moe_layer(x, idx, wt, bank, bank, down)
        return jq.mxfp4_gather_matmul(x, bank, rhs_indices=idx)

    want = use(jq.MXFP4ExpertBank(w, s), jq.MXFP4ExpertBank(w2, s2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bank, down = jq.MXFP4ExpertBank(w, s), jq.MXFP4ExpertBank(w2, s2)
        captured = use(bank, down)
    before = use(bank, down)                               # nothing of the capture has run
    assert bank.codes_tab.tolist() == [w.data_ptr() + e * N * K // 2 for e in range(E)]
    assert bank.scales_tab.tolist() == [s.data_ptr() + e * N * K // 32 for e in range(E)]
    graph.replay()
    after = use(bank, down)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        aside = use(bank, down)
    torch.cuda.synchronize()
    assert torch.equal(before, want) and torch.equal(captured, want) and torch.equal(after, want) and torch.equal(aside, want)
    del graph
    assert torch.equal(use(bank, down), want)


@pytest.mark.gpu
@pytest.mark.parametrize("E", [1550, 1551, 4097])
@pytest.mark.parametrize("T", [20, 90])
def test_banks_around_the_largest_sort(E, T):
    """Routed pairs of banks that the sort takes and of larger ones, whose pairs go one by one at any number.  Sums of 32 .. 64
    products of which each is a small multiple of 2^-4 are exact in float32; one rounding to bf16 follows."""
    N, K, k = 32, 64, 2
    rng = np.random.default_rng(E + T)
    words, byte = mo.pack(rng.integers(0, 16, (E, N, K)).astype(np.uint8)), np.full((E, N, K // 32), 126, np.uint8)
    w = mo.values(words, byte)
    bank = jq.MXFP4ExpertBank(torch.from_numpy(words.view(np.int32)).cuda(), torch.from_numpy(byte).cuda())
    x = torch.from_numpy(rng.integers(-4, 5, (T, K)) / 4.0).to(torch.bfloat16).cuda()
    idx = rng.integers(0, E, (T, k))
    idx[0], idx[1] = (0, E - 1), (E - 1, min(E - 1, 1550))
    ids = torch.from_numpy(idx).int().cuda()
    want = np.einsum("tk,tjnk->tjn", x.double().cpu().numpy(), w[idx])
    y = jq.mxfp4_gather_matmul(x, bank, rhs_indices=ids).reshape(T, k, N)
    assert torch.equal(y.cpu(), torch.from_numpy(want).to(torch.bfloat16))
    # the whole layer, I = 64: half a step each for g, u, h, the expert's row and (few pairs) the product of the first three, with
    # |silu'| <= 1.1 for what g does to h, and float32 sums far below
    down = jq.MXFP4ExpertBank.from_float(_rand(5, (E, 24, K), 0.1))
    gate = jq.MXFP4ExpertBank(bank.weight.repeat(1, 2, 1), bank.scales.repeat(1, 2, 1))
    out = jq.moe_layer(x, ids, torch.full((T, k), 0.5, device="cuda"), gate, gate, down, out_f32=True).double().cpu().numpy()
    d = mo.values(down.weight.cpu().numpy().view(np.uint32), down.scales.cpu().numpy())[idx]
    g = np.concatenate([want, want], -1)
    silu = g / (1.0 + np.exp(-g))
    h = 0.5 * silu * g
    spread = 2 * np.abs(h) + 0.5 * (1.1 * np.abs(g) + np.abs(silu)) * np.abs(g)
    ref, mag = np.einsum("tjk,tjnk->tn", h, d), np.einsum("tjk,tjnk->tn", spread + np.abs(h), np.abs(d))
    assert np.all(np.abs(out - ref) <= (2.0 ** -8 + 2.0 ** -14) * mag)


def test_largest_sort_is_the_library_s():
    lib, L = jq._lib.load(), jq._lib
    p, most = 1024, L.MOE_SORT_MAX_EXPERTS
    assert lib.jq_moe_sort(p, 64, most + 1, 0, p, p, p, 192, p, p, p, None) == L.JQ_EUNSUPPORTED
    assert lib.jq_moe_sort(p, 64, 0, 0, p, p, p, 192, p, p, p, None) == L.JQ_EUNSUPPORTED
    assert lib.jq_moe_sort(p, 64, most, 0, p, p, p, 0, p, p, p, None) == L.JQ_EINVAL         # only the tile is wrong
