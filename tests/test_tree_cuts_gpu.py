"""The tree attention where its forms meet: units of two row tiles that are cut, windows that are cut, blocks that pass from units of one tile to units
of two; accepted paths of masks that are no trees; keys and values written by the product on pairs of SMs beside their positions; steps of many
nodes and of many shapes."""

import numpy as np
import pytest
import torch

import helpers
import test_generate_gpu as generation
from tree_cases import TreeStep, signed
from test_tree_ops_gpu import accept_case, accept_run

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def ops():
    from boring_llm_b200.kernels import ops as o
    return o


@pytest.fixture(autouse=True)
def waits_ended():
    """No block has given up on a bounded wait."""
    yield
    ops().check_status()


def check(s, window=0):
    got = s.run(window)
    assert torch.equal(got, s.run(window))
    if window:                                                    # (the formula works on zeros where pages are gone)
        for t in (s.k, s.v):
            t[~torch.isfinite(t)] = 0.0
    s.check(got, window, probabilities_bf16=got.dtype == torch.bfloat16)


@pytest.mark.parametrize("masks,count,path", [
    ([0b1, 0b11, 0b101, 0b0111], 2, [0, 1]),                      # node 3 sees two children of node 0 and not itself
    ([0b1, 0b11, 0b111, 0b0111], 3, [0, 1, 2]),                   # ... and one that sees all of a path, but not itself
    ([0b1, 0b111, 0b101, 0b1101], 3, [0, 2, 3]),                  # node 1 sees itself and a later node
    ([0b1, 0b10, 0b110, 0b111], 1, [0]),                          # further roots
    ([0b1, 0b01, 0b01, 0b01], 1, [0])])
def test_a_node_that_does_not_see_itself_is_not_accepted(masks, count, path):
    """Every node holds the token that is sampled everywhere: only the masks decide."""
    s, tokens, sampled, k, v = accept_case([4], [13], 2, 64, 16, 2, torch.float32, 4)
    tokens[:], sampled[:] = 5, 5
    s.mask = torch.tensor(signed(masks), dtype=torch.int64)
    before = k.clone(), v.clone()
    counts, way, answer = accept_run(s, tokens, sampled, k, v)
    assert counts.tolist() == [count] and way[0].tolist() == path + [-1] * (64 - count) and answer[0].tolist() == [5] * count + [-1] * (64 - count)
    row = lambda t, i: t[:, int(s.table[0, (13 + i) // 16]), :, (13 + i) % 16]
    for j in range(4):
        node = path[j] if j < count else j
        assert torch.equal(row(k, j), row(before[0], node)) and torch.equal(row(v, j), row(before[1], node))
