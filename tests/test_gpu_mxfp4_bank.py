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
