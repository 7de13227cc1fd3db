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


def test_drafted_steps_of_many_requests_share_their_captured_shapes(model_folders):
    """Eight requests that draft as much as their text gives: a captured step for each padded number of nodes, and the right tokens."""
    from boring_llm_b200 import Engine
    d = model_folders("D", "bfloat16", 0.02)
    rng = np.random.default_rng(2)
    phrases = [helpers.random_tokens(300, 5, 70 + i) for i in range(4)]
    prompts = [sum((phrases[int(rng.integers(0, 4))] for _ in range(6 + i)), []) for i in range(8)]
    eng = Engine(d, dtype="bfloat16", ctx_size=256, max_num_seqs=8, max_tokens=2048, draft_tokens=31, debug_poison=True)
    got = eng.generate(prompts, n_predict=60, ignore_eos=True)
    for p, o in zip(prompts, got):
        assert len(o) == 60
        generation.check_greedy(d, p, o, "bfloat16")
    assert 0 < len(eng.runner._tree_graphs) <= 7 and eng.stats()["accepted_tokens"] > 0
    eng.runner.cache.check()


def tree_of(out, at, vocab, n):
    """n nodes: the certain token, a long wrong chain, and behind it the three right tokens."""
    wrong = (out[at + 1] + 1) % vocab
    tokens, parents = [out[at]] + [wrong] * (n - 4), [-1] + list(range(n - 4))
    return tokens + out[at + 1:at + 4], parents + [0, n - 3, n - 2]


@pytest.mark.parametrize("cuda_graphs", [True, False])
def test_steps_of_many_nodes(model_folders, cuda_graphs):
    """256 nodes and more: the product on pairs of SMs writes keys and values, the tree attention reads them, the right branch (the last one) is kept and its
    rows have moved: what is said afterwards is what the plain implementation says."""
    from boring_llm_b200 import Engine, StepEntry, TreeEntry
    from boring_llm_b200.sampling.params import SamplingParams, XorShift64
    d = model_folders("D", "bfloat16", 0.02)
    vocab = helpers.TINY["D"]["vocab_size"]
    run = Engine(d, dtype="bfloat16", ctx_size=512, max_num_seqs=8, max_tokens=4096, cuda_graphs=cuda_graphs).runner
    prompts = [helpers.random_tokens(vocab, 20 + 33 * i, 60 + i) for i in range(8)]
    truth = []
    for i, p in enumerate(prompts):
        out = [int(run.step([StepEntry(("t", i), p, [len(p) - 1])])[0].argmax())]
        while len(out) < 14:
            out.append(int(run.step([StepEntry(("t", i), [out[-1]], [0])])[0].argmax()))
        truth.append(out)
        run.free_request(("t", i))
        run.step([StepEntry(i, p, [])])
    said = [[t[0]] for t in truth]
    whole = 0
    for _ in range(3):
        entries = []
        for i in range(8):
            at = len(said[i]) - 1
            # (a request that has left the truth at a near tie goes on alone)
            tokens, parents = tree_of(truth[i], at, vocab, 40) if said[i] == truth[i][:at + 1] else ([said[i][-1]] * 40, [-1] + list(range(39)))
            entries.append(TreeEntry(i, tokens, parents))
        got = run.step_tree(entries, [(SamplingParams(), XorShift64(0), None)] * 8)
        for i in range(8):
            whole += len(got[i]) == 4
            said[i] += got[i][:4]
            run.truncate(i, len(prompts[i]) + len(said[i]) - 1)
    assert whole > 12                                             # most trees hold
    for i in range(8):
        said[i].append(int(run.step([StepEntry(i, [said[i][-1]], [0])])[0].argmax()))
        generation.check_greedy(d, prompts[i], said[i], "bfloat16")
    run.check_kernels()
    assert (run.graph_steps > 0) == cuda_graphs
